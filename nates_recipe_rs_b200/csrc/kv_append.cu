// Keys and values of new tokens into a paged cache, the rotary embedding applied on the way: the counterpart, for a batch of
// sequences at positions of their own, of the upstream's gpu_rope_partial (gpu-core/src/infer_ops.rs:61-83,
// gpu-core/src/kernels/f64_infer.hip:107-132: NeoX pairs (j, j + rotary_dim/2) of the first rotary_dim elements, angle
// pos * theta^(-2j/rotary_dim)) followed by the copy into the cache.
// Measured: 12122 tokens of 64/8 heads of 128, f32 to bf16: 122 us, 6.1 TB/s; 8 tokens 5.3 us.
// One pass: a row [q | k | v] is read once, the rotated queries go to q_out and k and v to their slots, all in the cache's type
// (one rounding from f32).  Bound by these bytes (many tokens) or by the latency of a launch (few).
// A CTA takes a few tokens.  It finds their sequences with one parallel read of cu_q, then computes each token's sines and
// cosines ONCE for all heads: the angle in f64 and reduced to [-pi, pi] there (at position 100000 an f32 angle is off by 4e-3),
// sine and cosine in f32.
#include "attn_pages.cuh"

namespace qmm {

constexpr int KVA_THREADS = 256;
constexpr int KVA_MAX_TOKENS = 8;   // per CTA
constexpr int KVA_MAX_PAIRS = 128;  // rotary_dim / 2

struct AppendParams {
    const void* qkv;
    void* q_out;
    void* k;
    void* v;
    const int* table;
    const int* cu_q;
    const int* kv_len;
    long qkv_stride, k_page, v_page;
    int table_stride, page_size, n_pages, n_seqs, total_q, max_kv;
    int nqh, nkv, hd, half, tokens;   // half: rotary_dim / 2; tokens per CTA
    double freq[KVA_MAX_PAIRS];       // theta^(-2j/rotary_dim)
};

// V consecutive elements as f32 / in the cache's type (addresses aligned to V elements)
template <typename T, int V> __device__ __forceinline__ void load_v(const T* src, float (&x)[V]) {
    if constexpr (V == 1) {
        x[0] = to_f32<T>(*src);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const float4 f = __ldcs(reinterpret_cast<const float4*>(src) + i);
            x[4 * i] = f.x, x[4 * i + 1] = f.y, x[4 * i + 2] = f.z, x[4 * i + 3] = f.w;
        }
    } else {
        static_assert(V == 8, "16 bytes");
        const uint4 u = __ldcs(reinterpret_cast<const uint4*>(src));
        const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(h[i]);
    }
}
template <typename T, int V> __device__ __forceinline__ void store_v(T* dst, const float (&x)[V]) {
    if constexpr (V == 1) {
        if constexpr (std::is_same<T, __half>::value) *dst = __float2half_rn(x[0]);
        else *dst = __float2bfloat16_rn(x[0]);
    } else {
        *reinterpret_cast<uint4*>(dst) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
    }
}

// TI: type of qkv, TO: type of the cache and of q_out, V: elements per access (8; 1 where half or hd is not a multiple of 8)
template <typename TI, typename TO, int V>
__global__ void __launch_bounds__(KVA_THREADS) rope_kv_append_paged_kernel(const __grid_constant__ AppendParams p) {
    __shared__ float2 turn[KVA_MAX_TOKENS][KVA_MAX_PAIRS];  // (cos, sin)
    __shared__ int count[KVA_MAX_TOKENS];
    __shared__ long long slot[KVA_MAX_TOKENS][2];           // element offset of the token's k and v slots, -1: none
    __shared__ int known[KVA_MAX_TOKENS];                   // the row belongs to a sequence
    const int tid = threadIdx.x, row0 = blockIdx.x * p.tokens, n = min(p.tokens, p.total_q - row0);
    if (tid < KVA_MAX_TOKENS) count[tid] = 0;
    pdl_wait_prior_grids();
    __syncthreads();
    // sequence of row r = how many of cu_q[1..n_seqs] are at most r
    int mine[KVA_MAX_TOKENS];
#pragma unroll
    for (int u = 0; u < KVA_MAX_TOKENS; ++u) mine[u] = 0;
    for (int s = tid + 1; s <= p.n_seqs; s += KVA_THREADS) {
        const int c = p.cu_q[s];
#pragma unroll
        for (int u = 0; u < KVA_MAX_TOKENS; ++u) mine[u] += c <= row0 + u;
    }
#pragma unroll
    for (int u = 0; u < KVA_MAX_TOKENS; ++u) {
        const int all = __reduce_add_sync(0xffffffffu, mine[u]);
        if ((tid & 31) == 0 && all) atomicAdd(&count[u], all);
    }
    __syncthreads();
    // position, angles and slots: a warp per token at a time
    for (int u = tid >> 5; u < n; u += KVA_THREADS / 32) {
        const int lane = tid & 31, s = count[u], r = row0 + u;
        const bool in = s < p.n_seqs && r >= p.cu_q[0];
        long pos = 0;
        if (in) {
            const int a = p.cu_q[s], b = p.cu_q[s + 1], kv = p.kv_len[s];
            pos = (long)kv - (b - a) + (r - a);
            const long cap = min((long)p.max_kv, (long)p.table_stride * p.page_size);
            const bool bad = kv < 0 || kv > cap || a < 0 || b > p.total_q;
            if (lane == 0) {
                long long ko = -1, vo = -1;
                if (bad) raise_status(DEV_BAD_LENGTH);
                if (pos >= 0 && pos < cap) {
                    const int id = p.table[(size_t)s * p.table_stride + pos / p.page_size];
                    if (id >= 0 && id < p.n_pages) {
                        const long long in_page = (long long)(pos % p.page_size) * p.nkv * p.hd;
                        ko = (long long)id * p.k_page + in_page, vo = (long long)id * p.v_page + in_page;
                    } else {
                        raise_status(DEV_BAD_PAGE);
                    }
                }
                slot[u][0] = ko, slot[u][1] = vo;
            }
        }
        if (lane == 0) known[u] = in;
        for (int j = lane; j < p.half; j += 32) {
            const double angle = (double)pos * p.freq[j];
            const double turns = rint(angle * 0.15915494309189533577);  // 1 / (2 pi)
            const float rest = (float)fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586232, angle));  // 2 pi in two parts
            float sn, cs;
            sincosf(rest, &sn, &cs);
            turn[u][j] = make_float2(cs, sn);
        }
    }
    __syncthreads();
    // work units of a token: V pairs of a q or k head; V elements of what is not rotated; V elements of v
    const int pu = p.half / V, ru = (p.hd - 2 * p.half) / V, hu = p.hd / V;
    const int qk = p.nqh + p.nkv, u_rot = qk * pu, u_rest = qk * ru, u_all = u_rot + u_rest + p.nkv * hu;
    const TI* qkv = static_cast<const TI*>(p.qkv);
    TO* q_out = static_cast<TO*>(p.q_out);
    TO* kp = static_cast<TO*>(p.k);
    TO* vp = static_cast<TO*>(p.v);
    for (int i = tid; i < n * u_all; i += KVA_THREADS) {
        const int u = i / u_all;
        int w = i - u * u_all;
        if (!known[u]) continue;  // rows of no sequence are left as they were
        const size_t r = (size_t)(row0 + u);
        const TI* row = qkv + r * p.qkv_stride;
        if (w < u_rot) {
            const int head = w / pu, j = (w - head * pu) * V;
            float a[V], b[V];
            load_v<TI, V>(row + (size_t)head * p.hd + j, a);
            load_v<TI, V>(row + (size_t)head * p.hd + p.half + j, b);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 t = turn[u][j + e];
                const float x = a[e] * t.x - b[e] * t.y, y = a[e] * t.y + b[e] * t.x;
                a[e] = x, b[e] = y;
            }
            TO* dst = nullptr;
            if (head < p.nqh) dst = q_out + (r * p.nqh + head) * p.hd;
            else if (slot[u][0] >= 0) dst = kp + slot[u][0] + (size_t)(head - p.nqh) * p.hd;
            if (dst) store_v<TO, V>(dst + j, a), store_v<TO, V>(dst + p.half + j, b);
        } else if (w < u_rot + u_rest) {
            w -= u_rot;
            const int head = w / ru, j = 2 * p.half + (w - head * ru) * V;
            float a[V];
            load_v<TI, V>(row + (size_t)head * p.hd + j, a);
            if (head < p.nqh) store_v<TO, V>(q_out + (r * p.nqh + head) * p.hd + j, a);
            else if (slot[u][0] >= 0) store_v<TO, V>(kp + slot[u][0] + (size_t)(head - p.nqh) * p.hd + j, a);
        } else if (slot[u][1] >= 0) {
            const int j = (w - u_rot - u_rest) * V;
            float a[V];
            load_v<TI, V>(row + (size_t)qk * p.hd + j, a);
            store_v<TO, V>(vp + slot[u][1] + j, a);
        }
    }
}

template <typename TI, typename TO>
static int kv_append_inst(const AppendParams& p, bool wide, cudaStream_t s) {
    const dim3 grid((p.total_q + p.tokens - 1) / p.tokens);
    return wide ? launch_overlapped(rope_kv_append_paged_kernel<TI, TO, 8>, grid, dim3(KVA_THREADS), 0, s, p)
                : launch_overlapped(rope_kv_append_paged_kernel<TI, TO, 1>, grid, dim3(KVA_THREADS), 0, s, p);
}

}  // namespace qmm
