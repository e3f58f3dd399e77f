// What the operators on a paged KV cache share: the view of a batch of sequences and of the cache, the tensor maps through
// which tiles of keys and values arrive, and what is done about values that are not finite under a mask.
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
constexpr int ATT_MAX_KEYS = 0x7FFFFFFF - 4095;  // positions of a tile past the last key, and of its up to 32 boxes, stay in 32 bits

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
// The first key that position pos sees (a position before 0 sees none: kept out of the difference, which a wide window would overflow)
__device__ __forceinline__ int first_key(const AttnParams& p, int pos) { return p.window ? max(max(pos, 0) - p.window + 1, 0) : 0; }
__device__ __forceinline__ KeyRange key_range(const AttnParams& p, const SeqInfo& si, int tok0, int tok1) {
    const int p0 = si.kv - si.q_len + tok0, p1 = si.kv - si.q_len + tok1 - 1;  // first and last position
    KeyRange r;
    r.a = first_key(p, p0);
    r.b = max(p1 + 1, 0);
    r.a2 = first_key(p, p1);
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
// The boxes of tile `t` (TILE positions) that hold a key of [a, b), the keys that some row sees: first, and how many.  What no box
// covers is whatever was there before: the reader clears the rows outside [a, b) (of the values; scores are masked).
template <int TILE>
__device__ __forceinline__ void tile_boxes(const AttnParams& p, int t, int a, int b, int& first, int& count) {
    const int lo = max(a - t * TILE, 0), hi = min(b - t * TILE, TILE);
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

// ---- values that are not finite under a mask ----
// The tensor cores add 0 * v for a masked key, which is not 0 when v is an infinity or a NaN.  So in the keys that some rows of an
// item see and others do not, such values are made zeros in shared memory (clean_value), and added to the outputs of the rows that
// do see them afterwards (add_odd_values): v + anything is v or NaN, whatever its weight, so no product is needed.
// Eight 16-bit values: those that are not finite become zeros; returns whether there were any
template <typename T> __device__ __forceinline__ bool odd_word(uint32_t w);  // of two values
template <> __device__ __forceinline__ bool odd_word<__half>(uint32_t w) { return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u; }
template <> __device__ __forceinline__ bool odd_word<__nv_bfloat16>(uint32_t w) { return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u; }
template <typename T> __device__ __forceinline__ uint32_t clean_word(uint32_t w) {
    constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
    if ((w & E) == E) w &= 0xFFFF0000u;
    if ((w & (E << 16)) == E << 16) w &= 0x0000FFFFu;
    return w;
}
template <typename T> __device__ __forceinline__ uint32_t times_zero(uint32_t w, uint32_t acc);  // acc + 0 * w: 0, or NaN
template <> __device__ __forceinline__ uint32_t times_zero<__half>(uint32_t w, uint32_t acc) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&w), __half2(__half(0.f), __half(0.f)), *reinterpret_cast<const __half2*>(&acc));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <> __device__ __forceinline__ uint32_t times_zero<__nv_bfloat16>(uint32_t w, uint32_t acc) {
    const __nv_bfloat162 z = __floats2bfloat162_rn(0.f, 0.f), r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w), z, *reinterpret_cast<const __nv_bfloat162*>(&acc));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// Rows [r0, r1) of one chunk of a value tile (8 pieces of 16 bytes a row): those outside [z0, z1) become zeros, the others are
// cleaned.  `threads` threads, this one number `i0`, U pieces in flight each.  Returns whether a value was made zero that some row
// sees.
template <typename T, int U>
__device__ __forceinline__ bool clear_values(uint4* chunk, int r0, int r1, int z0, int z1, int i0, int threads) {
    z0 = min(max(z0, r0), r1), z1 = min(max(z1, z0), r1);
#pragma unroll 4
    for (int i = r0 * 8 + i0; i < z0 * 8; i += threads) chunk[i] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 4
    for (int i = z1 * 8 + i0; i < r1 * 8; i += threads) chunk[i] = make_uint4(0u, 0u, 0u, 0u);
    bool odd = false;
#pragma unroll 1
    for (int b = z0 * 8 + i0; b < z1 * 8; b += U * threads) {
        uint4 y[U];
#pragma unroll
        for (int u = 0; u < U; ++u) y[u] = b + u * threads < z1 * 8 ? chunk[b + u * threads] : make_uint4(0u, 0u, 0u, 0u);
        uint32_t a0 = 0u, a1 = 0u, a2 = 0u, a3 = 0u;
#pragma unroll
        for (int u = 0; u < U; ++u)
            a0 = times_zero<T>(y[u].x, a0), a1 = times_zero<T>(y[u].y, a1), a2 = times_zero<T>(y[u].z, a2), a3 = times_zero<T>(y[u].w, a3);
        if (!(odd_word<T>(a0) || odd_word<T>(a1) || odd_word<T>(a2) || odd_word<T>(a3))) continue;
        odd = true;
#pragma unroll 1
        for (int i = b; i < min(b + U * threads, z1 * 8); i += threads) {
            uint4 x = chunk[i];
            x.x = clean_word<T>(x.x), x.y = clean_word<T>(x.y), x.z = clean_word<T>(x.z), x.w = clean_word<T>(x.w);
            chunk[i] = x;
        }
    }
    return odd;
}
__device__ __forceinline__ float load_out1(const void* out, int dtype, size_t e) {
    return dtype == QMM_DT_F32 ? static_cast<const float*>(out)[e] : dtype == QMM_DT_F16 ? __half2float(static_cast<const __half*>(out)[e])
                                                                                         : __bfloat162float(static_cast<const __nv_bfloat16*>(out)[e]);
}
// Keys [k0, k1) of sequence s, rows [r0, r1) of its (token, head of the group) list: adds the values that are not finite to the
// outputs of the rows that see them, as stored in `out` (so null) or in a part so of which row `so_row` is the first.  One warp,
// after its own stores to these rows.
template <typename T, int HD>
__device__ __noinline__ void add_odd_values(const AttnParams& p, int s, int q0, int pos0, int kvh, int k0, int k1, int r0, int r1, float* so, int so_row) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll 1
    for (int key = k0; key < k1; ++key) {
        size_t vo;
        if (p.table) {
            const int pg = page_of(p, s, key / p.page_size);
            if (pg >= p.n_pages) continue;
            vo = (size_t)pg * p.v_page + (size_t)(key % p.page_size) * p.v_row;
        } else {
            vo = (size_t)(q0 + key) * p.v_row;
        }
        const T* vr = static_cast<const T*>(p.v) + vo + (size_t)kvh * HD;
        float v[HD / 32];
        bool odd = false;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) v[j] = to_f32<T>(vr[lane + 32 * j]), odd |= v[j] * 0.f != 0.f;
        if (!__any_sync(0xffffffffu, odd)) continue;
#pragma unroll 1
        for (int r = r0; r < r1; ++r) {
            const int tok = r / p.group, pos = pos0 + tok;
            if (key > pos || (p.window && key <= pos - p.window)) continue;
            const size_t e = (size_t)(q0 + tok) * p.out_stride + (size_t)(kvh * p.group + r - tok * p.group) * HD + lane;
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) {
                if (v[j] * 0.f == 0.f) continue;
                if (so) so[(size_t)(r - so_row) * HD + lane + 32 * j] += v[j];
                else store_out1(p.out, p.out_dtype, e + 32 * j, load_out1(p.out, p.out_dtype, e + 32 * j) + v[j]);
            }
        }
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
