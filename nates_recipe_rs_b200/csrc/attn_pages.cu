// Entry points of the operators on a paged KV cache and on packed prompts (declared in include/qmm.h): argument checks, tensor
// maps and the choice of kernel.
#include "attn_pages.cuh"
#include <algorithm>
#include <cmath>

namespace qmm {

int kv_tensor_map(CUtensorMap* map, const void* base, int dtype, int hd, int nkv, long rows, long n_pages, long row_stride, long page_stride,
                  int box_rows) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return cuda_fail(cudaErrorNotSupported);
    const cuuint64_t dims[4] = {(cuuint64_t)hd, (cuuint64_t)nkv, (cuuint64_t)rows, (cuuint64_t)n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)hd * 2, (cuuint64_t)row_stride * 2, (cuuint64_t)page_stride * 2};
    const cuuint32_t box[4] = {64, 1, (cuuint32_t)box_rows, 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    if (enc(map, dtype == QMM_DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides,
            box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cuda_fail(cudaErrorInvalidValue);
    return QMM_OK;
}

static int gcd_int(int a, int b) {
    while (b) {
        const int c = a % b;
        a = b, b = c;
    }
    return a;
}
static bool misaligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

static int check_batch(const qmm_seq_batch* b, bool with_kv) {
    if (!b || !b->cu_q || (with_kv && !b->kv_len)) return QMM_ERR_NULL;
    if (b->n_seqs <= 0 || b->total_q < 0 || b->max_q < 0 || (with_kv && b->max_kv < 0)) return QMM_ERR_SHAPE;
    if (b->n_seqs > ATT_MAX_SEQS) return QMM_ERR_UNSUPPORTED;
    return QMM_OK;
}
// The pool of a paged cache; fills in the page strides
static int check_pool(const qmm_paged_kv* kv, long& k_page, long& v_page) {
    if (!kv || !kv->k_pages || !kv->v_pages || !kv->page_table) return QMM_ERR_NULL;
    if (kv->dtype != QMM_DT_F16 && kv->dtype != QMM_DT_BF16) return QMM_ERR_TYPE;
    if (kv->n_pages <= 0 || kv->page_size <= 0 || kv->n_kv_heads <= 0 || kv->head_dim <= 0 || kv->table_stride < 0 || kv->k_page_stride < 0 ||
        kv->v_page_stride < 0)
        return QMM_ERR_SHAPE;
    const long page = (long)kv->page_size * kv->n_kv_heads * kv->head_dim;
    k_page = kv->k_page_stride ? kv->k_page_stride : page;
    v_page = kv->v_page_stride ? kv->v_page_stride : page;
    if (k_page < page || v_page < page) return QMM_ERR_SHAPE;
    if (misaligned(kv->k_pages, 16) || misaligned(kv->v_pages, 16) || k_page % 8 || v_page % 8) return QMM_ERR_ALIGN;
    return QMM_OK;
}
static int check_heads(int nqh, int nkv, int hd) {
    if (nqh <= 0 || nkv <= 0 || hd <= 0 || nqh % nkv) return QMM_ERR_SHAPE;
    if (nqh / nkv > ATT_MAX_GROUP || nkv > 65535 || (hd != 32 && hd != 64 && hd != 96 && hd != 128 && hd != 256)) return QMM_ERR_UNSUPPORTED;
    return QMM_OK;
}
static int check_out(const void* out, int dtype, long stride, int nqh, int hd) {
    if (!out) return QMM_ERR_NULL;
    if (dtype != QMM_DT_F16 && dtype != QMM_DT_BF16 && dtype != QMM_DT_F32) return QMM_ERR_TYPE;
    if (stride < (long)nqh * hd) return QMM_ERR_SHAPE;
    if (misaligned(out, dtype == QMM_DT_F32 ? 8 : 4) || stride % 2) return QMM_ERR_ALIGN;
    return QMM_OK;
}
constexpr float LOG2_E = 1.4426950408889634f;  // weights are computed as exp2(x log2(e))
static bool bad_scale(float s) { return !(s > 0.f) || std::isinf(s * LOG2_E); }

// Up to 16 (token, query head of the group) rows per sequence and kv head: decode, bound by the cache (attn_rows.cu); more rows:
// the tcgen05 form (attn_tiles.cu), whose tiles of 128 rows are mostly empty below that.  Measured, us in attn_rows / attn_tiles,
// 64 sequences of 1000 to 7300 tokens, f16: 32/8 heads of 128, 1 token (4 rows) 178 / 227, 4 tokens (16 rows) 186 / 231, 5 tokens
// (20 rows) 342 / 232; 1 token of 34/2 heads (17 rows) 81 / 75.  Heads of 64 cross later (8/2 heads: 16 rows 37 / 66, 20 rows
// 56 / 67), heads of 256 a little earlier (4 rows 96 / 102, 16 rows 115 / 105).
static bool attn_narrow(long max_q, int group) { return max_q * group <= AR_ROWS; }
static int attn_run(bool narrow, AttnParams& p, int dtype, int hd, long rows, long n_pages, cudaStream_t s) {
    const int tile = narrow ? AR_TILE : AT_TILE;
    const int box = p.table ? gcd_int(p.page_size, tile) : tile;  // pages are multiples of 8, tiles powers of two
    for (p.box_shift = 3; 1 << p.box_shift < box;) ++p.box_shift;
    p.group_inv = (65536 + p.group - 1) / p.group;
    p.row_tiles = attn_tiles_rows(hd) / 128;
    CUtensorMap km, vm;
    if (int st = kv_tensor_map(&km, p.k, dtype, hd, p.nkv, rows, n_pages, p.k_row, p.k_page, box)) return st;
    if (int st = kv_tensor_map(&vm, p.v, dtype, hd, p.nkv, rows, n_pages, p.v_row, p.v_page, box)) return st;
    return narrow ? attn_rows_launch(p, km, vm, dtype, hd, s) : attn_tiles_launch(p, km, vm, dtype, hd, s);
}

}  // namespace qmm

using namespace qmm;

extern "C" {

int launch_rope_kv_append_paged(const void* qkv, int qkv_dtype, long qkv_stride, void* q_out, const qmm_paged_kv* kv, const qmm_seq_batch* seqs,
                                int n_q_heads, int rotary_dim, float theta, void* stream) {
    AppendParams p = {};
    if (!qkv || !q_out) return QMM_ERR_NULL;
    if (int st = check_batch(seqs, true)) return st;
    if (int st = check_pool(kv, p.k_page, p.v_page)) return st;
    if (qkv_dtype != QMM_DT_F32 && qkv_dtype != QMM_DT_F16 && qkv_dtype != QMM_DT_BF16) return QMM_ERR_TYPE;
    const int hd = kv->head_dim, nkv = kv->n_kv_heads;
    const long row = ((long)n_q_heads + 2l * nkv) * hd;
    if (n_q_heads <= 0 || rotary_dim < 0 || rotary_dim % 2 || rotary_dim > hd || qkv_stride < row || !(theta > 0.f) || std::isinf(theta))
        return QMM_ERR_SHAPE;
    if (rotary_dim > 2 * KVA_MAX_PAIRS || hd > 1024 || row > 1 << 22) return QMM_ERR_UNSUPPORTED;
    const int size_in = qkv_dtype == QMM_DT_F32 ? 4 : 2;
    if (misaligned(qkv, size_in) || misaligned(q_out, 2)) return QMM_ERR_ALIGN;
    if (qkv == q_out) return QMM_ERR_SHAPE;
    if (seqs->total_q == 0) return QMM_OK;
    p.qkv = qkv, p.q_out = q_out, p.k = const_cast<void*>(kv->k_pages), p.v = const_cast<void*>(kv->v_pages);
    p.table = kv->page_table, p.cu_q = seqs->cu_q, p.kv_len = seqs->kv_len;
    p.qkv_stride = qkv_stride;
    p.table_stride = kv->table_stride, p.page_size = kv->page_size, p.n_pages = kv->n_pages;
    p.n_seqs = seqs->n_seqs, p.total_q = seqs->total_q, p.max_kv = seqs->max_kv;
    p.nqh = n_q_heads, p.nkv = nkv, p.hd = hd, p.half = rotary_dim / 2;
    const double step = rotary_dim ? std::pow((double)theta, -2.0 / rotary_dim) : 1.0;
    p.freq[0] = 1.0;  // (127 products in f64 are off by at most 127 * 2^-53 relative)
    for (int j = 1; j < p.half; ++j) p.freq[j] = p.freq[j - 1] * step;
    // 16-byte accesses where every head, half head and row begins on one
    const bool wide = p.half % 8 == 0 && hd % 8 == 0 && !misaligned(qkv, 16) && !misaligned(q_out, 16) && qkv_stride * size_in % 16 == 0;
    // As few CTAs as run at once (six per SM), so that what a CTA does before its first byte (finding the sequences, the angles) is
    // not paid in two rounds: 2431 tokens of 20 heads of 96 take 7.6 us with three tokens per CTA, 11.2 with one; but no more work
    // than twice what its threads take at a time, or two tokens: 12122 tokens of 80 heads of 128 take 121 us with two, 131 with eight
    const long units = row / 16, at_once = 6l * sm_count();
    const long most = std::min<long>(KVA_MAX_TOKENS, std::max<long>(2, 2 * KVA_THREADS / std::max<long>(units, 1)));
    p.tokens = (int)std::min(most, std::max<long>(1, (seqs->total_q + at_once - 1) / at_once));
    cudaStream_t s = as_stream(stream);
    const bool f16 = kv->dtype == QMM_DT_F16;
    if (qkv_dtype == QMM_DT_F32) return f16 ? kv_append_inst<float, __half>(p, wide, s) : kv_append_inst<float, __nv_bfloat16>(p, wide, s);
    if (qkv_dtype == QMM_DT_F16) return f16 ? kv_append_inst<__half, __half>(p, wide, s) : kv_append_inst<__half, __nv_bfloat16>(p, wide, s);
    return f16 ? kv_append_inst<__nv_bfloat16, __half>(p, wide, s) : kv_append_inst<__nv_bfloat16, __nv_bfloat16>(p, wide, s);
}

long qmm_attn_paged_scratch_bytes(int max_q, int n_q_heads, int n_kv_heads, int head_dim) {
    if (max_q < 0) return QMM_ERR_SHAPE;
    if (int st = check_heads(n_q_heads, n_kv_heads, head_dim)) return st;
    return attn_narrow(max_q, n_q_heads / n_kv_heads) ? attn_rows_scratch_bytes(head_dim) : attn_tiles_scratch_bytes(head_dim);
}

int launch_attn_paged(const void* q, long q_stride, const qmm_paged_kv* kv, const qmm_seq_batch* seqs, void* out, int out_dtype, long out_stride,
                      void* scratch, long scratch_bytes, int n_q_heads, int window, float kq_scale, void* stream) {
    AttnParams p = {};
    if (!q || !scratch) return QMM_ERR_NULL;
    if (int st = check_batch(seqs, true)) return st;
    if (int st = check_pool(kv, p.k_page, p.v_page)) return st;
    const int hd = kv->head_dim, nkv = kv->n_kv_heads;
    if (int st = check_heads(n_q_heads, nkv, hd)) return st;
    if (int st = check_out(out, out_dtype, out_stride, n_q_heads, hd)) return st;
    if (q_stride < (long)n_q_heads * hd || window < 0 || bad_scale(kq_scale) || out == q) return QMM_ERR_SHAPE;
    if (kv->page_size % 8) return QMM_ERR_UNSUPPORTED;
    if (misaligned(q, 16) || q_stride % 8 || misaligned(scratch, 16)) return QMM_ERR_ALIGN;
    if (scratch_bytes < qmm_attn_paged_scratch_bytes(seqs->max_q, n_q_heads, nkv, hd)) return QMM_ERR_SCRATCH;
    if (seqs->total_q == 0) return QMM_OK;
    p.q = q, p.k = kv->k_pages, p.v = kv->v_pages, p.out = out;
    p.table = kv->page_table, p.cu_q = seqs->cu_q, p.kv_len = seqs->kv_len, p.scratch = static_cast<float*>(scratch);
    p.q_stride = q_stride, p.out_stride = out_stride, p.k_row = p.v_row = (long)nkv * hd;
    p.table_stride = kv->table_stride, p.page_size = kv->page_size, p.n_pages = kv->n_pages;
    p.n_seqs = seqs->n_seqs, p.total_q = seqs->total_q, p.max_kv = std::min(seqs->max_kv, ATT_MAX_KEYS);
    p.nqh = n_q_heads, p.nkv = nkv, p.group = n_q_heads / nkv, p.window = window, p.out_dtype = out_dtype;
    p.scale_log2 = kq_scale * LOG2_E;
    // More rows: where their items would not fill the GPU several times over, their tiles are shared evenly, as those of decode
    // always are.  The host knows the rows and not the lengths.  Measured, us whole / shared (32/8 heads of 128, f16): 912 new tokens
    // on 8k and 16k 279 / 214, 512 on 32k 529 / 279 (shared); 100 x 60 on 1k 162 / 178, one prompt of 8000 494 / 932 (whole).  Not
    // seen by the rule: a prompt without a past, whose items see part of the tiles that sharing counts for them (2000 tokens 51 / 99,
    // 4000 tokens 144 / 268, shared), and one sequence far longer than the others (100 x 60 on 1k, one of them on 30k 621 / 205, whole).
    const bool narrow = attn_narrow(seqs->max_q, p.group);
    p.stream_k = ((long)p.total_q * p.group / attn_tiles_rows(hd) + 1) * nkv < 4l * sm_count();
    return attn_run(narrow, p, kv->dtype, hd, p.page_size, p.n_pages, as_stream(stream));
}

int launch_attn_packed(const void* q, const void* k, const void* v, int dtype, long q_stride, long k_stride, long v_stride,
                       const qmm_seq_batch* seqs, void* out, int out_dtype, long out_stride, int n_q_heads, int n_kv_heads, int head_dim, int window,
                       float kq_scale, void* stream) {
    AttnParams p = {};
    if (!q || !k || !v) return QMM_ERR_NULL;
    if (int st = check_batch(seqs, false)) return st;
    if (dtype != QMM_DT_F16 && dtype != QMM_DT_BF16) return QMM_ERR_TYPE;
    const int hd = head_dim, nkv = n_kv_heads;
    if (int st = check_heads(n_q_heads, nkv, hd)) return st;
    if (int st = check_out(out, out_dtype, out_stride, n_q_heads, hd)) return st;
    if (q_stride < (long)n_q_heads * hd || k_stride < (long)nkv * hd || v_stride < (long)nkv * hd || window < 0 || bad_scale(kq_scale) || out == q ||
        out == k || out == v)
        return QMM_ERR_SHAPE;
    if (misaligned(q, 16) || misaligned(k, 16) || misaligned(v, 16) || q_stride % 8 || k_stride % 8 || v_stride % 8) return QMM_ERR_ALIGN;
    if (seqs->total_q == 0) return QMM_OK;
    p.q = q, p.k = k, p.v = v, p.out = out;
    p.cu_q = seqs->cu_q;
    p.q_stride = q_stride, p.out_stride = out_stride, p.k_row = k_stride, p.v_row = v_stride;
    p.n_seqs = seqs->n_seqs, p.total_q = seqs->total_q, p.max_kv = seqs->max_q;
    p.nqh = n_q_heads, p.nkv = nkv, p.group = n_q_heads / nkv, p.window = window, p.out_dtype = out_dtype;
    p.scale_log2 = kq_scale * LOG2_E;
    p.k_page = (long)p.total_q * k_stride, p.v_page = (long)p.total_q * v_stride;  // one page of all rows
    return attn_run(false, p, dtype, hd, p.total_q, 1, as_stream(stream));
}

}  // extern "C"
