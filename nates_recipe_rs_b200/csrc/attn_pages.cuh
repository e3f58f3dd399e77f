// What the operators on a paged KV cache share: the view of a batch of sequences and of the cache, the tensor maps through
// which tiles of keys and values arrive, and the exact (slow) attention of one row.
//
// A batch is packed: the new tokens of sequence s are rows cu_q[s] .. cu_q[s+1]-1; row i of them is position
// kv_len[s] - q_len + i.  Position t of a sequence lies in page table[s][t / page_size], slot t % page_size.  A packed
// prompt without a cache is the same with ONE page of all rows: position t of sequence s is row cu_q[s] + t.
#pragma once
#include "qmm_formats.cuh"
#include <cuda.h>
#include <mutex>

namespace qmm {

constexpr int ATT_MAX_GROUP = 64;   // query heads of one kv head
constexpr int ATT_MAX_SEQS = 1 << 20;

struct AttnParams {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    const int* table;  // null: packed rows
    const int* cu_q;
    const int* kv_len;
    float* scratch;
    long q_stride, out_stride;               // elements between rows
    long k_row, v_row, k_page, v_page;       // elements between the slots of a page, and between pages
    int table_stride, page_size, n_pages;
    int n_seqs, total_q, max_kv;
    int nqh, nkv, group, window, out_dtype;
    int box_shift;                           // rows of one tensor-map box: 1 << box_shift, divides the tile and the page
    int row_tiles;                           // attn_tiles.cu: tiles of 128 rows of an item
    int group_inv;                           // ceil(2^16 / group): r / group = r * group_inv >> 16 for the rows r < 256 of an item
    int stream_k;                            // 1: the CTAs share all (item, tile) pairs evenly and joined items go through scratch
    float scale_log2;                        // kq_scale * log2(e)
};

struct SeqInfo {
    int q0, q_len, kv;  // first row, rows, keys
};

__device__ __forceinline__ void raise_status(int code) { atomicExch(&g_device_status, code); }

// A bounded wait whose first probe alone is inlined: these kernels wait in many places, and their code has to fit the
// instruction cache (items of a few tiles spent most of their time fetching code when everything was inlined and unrolled).
// Where the wait runs out the CTA's abort flag is set and the status raised.
__device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t parity, int code, volatile int* cta_abort) {
    if (mbar_wait_bounded(bar, parity, cta_abort)) return true;
    if (!*cta_abort) {
        raise_status(code);
        *cta_abort = 1;
    }
    return false;
}
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, int code, volatile int* cta_abort) {
    return mbar_try_wait(smem_u32(bar), parity) || wait_slow(smem_u32(bar), parity, code, cta_abort);
}

// The lengths of a sequence, held inside the buffers whatever the arrays say (a value outside raises the device status).
__device__ __noinline__ SeqInfo seq_info(const AttnParams& p, int s) {
    const int a = p.cu_q[s], b = p.cu_q[s + 1];
    SeqInfo r;
    r.q0 = min(max(a, 0), p.total_q);
    const int e = min(max(b, r.q0), p.total_q);
    r.q_len = e - r.q0;
    bool bad = r.q0 != a || e != b;
    if (p.table) {
        const int kv = p.kv_len[s];
        const long cap = min((long)p.max_kv, (long)p.table_stride * p.page_size);
        r.kv = (int)min((long)max(kv, 0), cap);
        bad |= r.kv != kv;
    } else {
        r.kv = r.q_len;
    }
    if (bad) raise_status(DEV_BAD_LENGTH);
    return r;
}

// Rows [r0, r1) of a sequence (r = token * group + head of the group): the keys any of them sees are [a, b), those all of
// them see [a2, b2) (empty ranges have a >= b).
struct KeyRange {
    int a, b, a2, b2;
};
__device__ __forceinline__ KeyRange key_range(const AttnParams& p, const SeqInfo& si, int tok0, int tok1) {
    const int p0 = si.kv - si.q_len + tok0, p1 = si.kv - si.q_len + tok1 - 1;  // first and last position
    KeyRange r;
    r.a = p.window ? max(0, p0 - p.window + 1) : 0;
    r.b = max(p1 + 1, 0);
    r.a2 = p.window ? max(0, p1 - p.window + 1) : 0;
    r.b2 = max(p0 + 1, 0);
    return r;
}

// Page of a position (n_pages, past the end, where the table holds no page: its rows arrive as zeros and the status is raised).
__device__ __forceinline__ int page_of(const AttnParams& p, int s, int page_idx) {
    const int id = p.table[(size_t)s * p.table_stride + page_idx];
    if (id < 0 || id >= p.n_pages) {
        raise_status(DEV_BAD_PAGE);
        return p.n_pages;
    }
    return id;
}

// Block-wide search: F::count(p, s) >= 0 items per sequence; finds the sequence that holds item `target` of all of them and the items
// before it.  Every thread of the block calls it; sh: 36 words.  Returns -1 when there are fewer items (total in `before`).
template <typename F>
__device__ __noinline__ int find_item(const AttnParams& p, long target, long& before, long long* sh) {
    const int n_seqs = p.n_seqs;
    const int nt = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = nt >> 5;
    long base = 0;
    int found = -1;
    long found_before = 0;
#pragma unroll 1
    for (int s0 = 0; s0 < n_seqs; s0 += nt) {
        const int s = s0 + threadIdx.x;
        const long long v = s < n_seqs ? (long long)F::count(p, s) : 0ll;
        long long inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        if (lane == 31) sh[warp] = inc;
        if (threadIdx.x == 0) sh[32] = -1;
        __syncthreads();
        long long wbase = base, all = 0;
#pragma unroll 1
        for (int w = 0; w < nw; ++w) {
            if (w < warp) wbase += sh[w];
            all += sh[w];
        }
        const long long excl = wbase + inc - v;
        if (target >= excl && target < excl + v) sh[32] = s, sh[33] = excl;
        __syncthreads();
        if (sh[32] >= 0) found = (int)sh[32], found_before = sh[33];
        base += all;
        __syncthreads();
        if (found >= 0) break;
    }
    before = found >= 0 ? found_before : base;
    return found;
}

// As find_item, by one warp: 32 sequences at a time
template <typename F>
__device__ __noinline__ int warp_find_item(const AttnParams& p, long target, long& before) {
    const int lane = threadIdx.x & 31;
    before = 0;
#pragma unroll 1
    for (int base = 0; base < p.n_seqs; base += 32) {
        const long long cnt = base + lane < p.n_seqs ? (long long)F::count(p, base + lane) : 0ll;
        long long inc = cnt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        const unsigned past = __ballot_sync(0xffffffffu, before + inc > target);
        if (past) {
            const int f = __ffs(past) - 1;
            before += __shfl_sync(0xffffffffu, inc - cnt, f);
            return base + f;
        }
        before += __shfl_sync(0xffffffffu, inc, 31);
    }
    return -1;
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two neighbouring outputs (element index e, even) in the output's type
__device__ __forceinline__ void store_out2(void* out, int dtype, size_t e, float a, float b) {
    if (dtype == QMM_DT_F32) *reinterpret_cast<float2*>(static_cast<float*>(out) + e) = make_float2(a, b);
    else if (dtype == QMM_DT_F16) *reinterpret_cast<uint32_t*>(static_cast<__half*>(out) + e) = pack2<__half>(a, b);
    else *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(out) + e) = pack2<__nv_bfloat16>(a, b);
}
__device__ __forceinline__ void store_out1(void* out, int dtype, size_t e, float a) {
    if (dtype == QMM_DT_F32) static_cast<float*>(out)[e] = a;
    else if (dtype == QMM_DT_F16) static_cast<__half*>(out)[e] = __float2half_rn(a);
    else static_cast<__nv_bfloat16*>(out)[e] = __float2bfloat16_rn(a);
}

// ---- tiles of keys and values ----
// One tensor map per matrix: (element, kv head, slot, page), boxes of 64 elements x box_rows slots, 128-byte swizzle.  A tile
// in shared memory is ceil(HD / 64) chunks of TILE rows x 128 bytes; elements past HD and rows of a missing page are zeros.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int h, int r, int pg, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(h), "r"(r), "r"(pg), "r"(bar)
                 : "memory");
}
// The boxes of tile `t` (TILE positions) that hold a key of [a, kv): first, and how many.  What no box covers, and what lies past
// kv in the last one, is whatever was there before: the reader clears those rows (of the values; scores are masked).
template <int TILE>
__device__ __forceinline__ void tile_boxes(const AttnParams& p, int t, int a, int kv, int& first, int& count) {
    const int lo = max(a - t * TILE, 0), hi = min(kv - t * TILE, TILE);
    first = lo >> p.box_shift;
    count = hi > lo ? ((hi - 1) >> p.box_shift) - first + 1 : 0;
}
// Issued by a whole warp: the boxes of one matrix's tile, elements from x0 on.  `pages` holds, in lane j, the page of box j (page_of_boxes).
template <int TILE, int NCH>
__device__ __forceinline__ void load_tile(const AttnParams& p, const CUtensorMap* map, uint32_t dst, uint32_t bar, int x0, int first, int count,
                                          int pages, int slots, int kvh) {
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int i = lane; i - lane < count * NCH; i += 32) {  // (the whole warp stays in the loop: the shuffles need it)
        const int j = first + i / NCH, c = i % NCH;
        const int pg = __shfl_sync(0xffffffffu, pages, j & 31), slot = __shfl_sync(0xffffffffu, slots, j & 31);
        if (i < count * NCH) tma_load_4d(dst + (uint32_t)(c * TILE + (j << p.box_shift)) * 128u, map, x0 + c * 64, kvh, slot, pg, bar);
    }
}
// lane j: page and slot of the first position of box j of tile t (looked up ahead of the tile's turn); packed rows are one page
template <int TILE>
__device__ __forceinline__ int page_of_boxes(const AttnParams& p, int s, int row0, int t, int first, int count, int& slot) {
    const int lane = threadIdx.x & 31, pos = t * TILE + (lane << p.box_shift);
    slot = row0 + pos;
    if (!p.table || lane < first || lane >= first + count) return 0;
    const int idx = pos / p.page_size;
    slot = pos - idx * p.page_size;
    return page_of(p, s, idx);
}

// ---- one row, exactly by the formula: keys [k0, k1) of those the row sees, one warp, lane l holds elements l + 32 j ----
// The tensor cores add 0 * v for a masked key, which is not 0 when v is an infinity or a NaN: rows whose output is not finite are
// computed again this way (where that is what the formula gives, it stays).  m is in units of the raw score.
template <typename T, int HD>
__device__ __noinline__ void attn_row_exact(const AttnParams& p, int s, int q0, int tok, int head, int kvh, int k0, int k1, float& m, float& l,
                                            float (&o)[HD / 32]) {
    const int lane = threadIdx.x & 31;
    const T* qr = static_cast<const T*>(p.q) + (size_t)(q0 + tok) * p.q_stride + (size_t)head * HD;
    float qv[HD / 32];
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) qv[j] = to_f32<T>(qr[lane + 32 * j]), o[j] = 0.f;
    m = -INFINITY, l = 0.f;
#pragma unroll 1
    for (int key = k0; key < k1; ++key) {
        size_t ko, vo;
        bool there = true;
        if (p.table) {
            const int pg = page_of(p, s, key / p.page_size), slot = key % p.page_size;
            there = pg < p.n_pages;
            ko = (size_t)pg * p.k_page + (size_t)slot * p.k_row, vo = (size_t)pg * p.v_page + (size_t)slot * p.v_row;
        } else {
            ko = (size_t)(q0 + key) * p.k_row, vo = (size_t)(q0 + key) * p.v_row;
        }
        const T* kr = static_cast<const T*>(p.k) + ko + (size_t)kvh * HD;
        const T* vr = static_cast<const T*>(p.v) + vo + (size_t)kvh * HD;
        float d = 0.f;
        if (there) {
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) d += qv[j] * to_f32<T>(kr[lane + 32 * j]);
        }
        d = warp_sum(d);
        const float mn = fmaxf(m, d), mu = mn == -INFINITY ? 0.f : mn;
        const float f = fast_exp2((m - mu) * p.scale_log2), e = fast_exp2((d - mu) * p.scale_log2);
        m = mn;
        l = l * f + e;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) o[j] = o[j] * f + (there ? e * to_f32<T>(vr[lane + 32 * j]) : 0.f);
    }
}

// ---- host side ----
// A launch that may begin while the kernel before it drains (its own first instruction that touches memory waits for that
// kernel), where the library's overlap setting allows it.
template <typename... KArgs, typename... Args>
static int launch_overlapped(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = overlap_enabled() ? 1 : 0;
    cfg.attrs = attr, cfg.numAttrs = 1;
    QMM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, args...));
    return QMM_OK;
}
int kv_tensor_map(CUtensorMap* map, const void* base, int dtype, int hd, int nkv, long rows, long n_pages, long row_stride, long page_stride,
                  int box_rows);

}  // namespace qmm
