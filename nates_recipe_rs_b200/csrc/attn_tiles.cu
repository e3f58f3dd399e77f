// Attention of many rows over a paged cache or over packed prompts on tcgen05: pieces of prompts and whole prompts.  Same
// operator and same conventions as attn_rows.cu.
//
// A CTA owns up to two tiles of 128 rows of one kv head; a row is a (token, query head of the group) pair, tokens outermost, so
// one tile of keys and values serves every query head that shares it and a tile spans few positions (128 / group tokens: little
// of the causal triangle is computed and thrown away).  For every tile of 128 keys and each of the two row tiles
//     S = Q K^T    128 x 128 x HD, both operands in shared memory, S in tensor memory (f32)
//     P = exp2((S - m) * c), row sums            in registers, S read with tcgen05.ld, P written back over S (16 bit)
//     O += P V     128 x HD x 128, P from tensor memory, V from shared memory as it arrives (keys are the K dimension: the
//                  operand is "MN major"), O in tensor memory for the whole run over the keys
// While the threads of one row tile compute exponentials the tensor cores work for the other: the two pipes (16 exponentials per
// clock and SM; 8192 flops) need about the same time at HD = 128, 2048 cycles per tile of keys, and so does shared memory (the
// operands of S = Q K^T alone take its whole bandwidth).  A step takes about 3600 cycles: scores, softmax and outputs of ONE row
// tile follow one another, and the turns (below) leave gaps.  Measured: 8192 tokens, 32/8 heads of 128, causal: 537 us in a
// graph replayed with pauses, 1020 TFLOP/s of the products that are not masked; 4096 tokens 155 us.  The running maximum that P is
// scaled by is only moved when a row's maximum has grown by more than 2^8 (P <= 256 fits f16, l and O are f32): O is rescaled in
// tensor memory a few times per run instead of once per tile, with no separate correction step.
// Warps: 0-7 and 8-15 softmax of row tile 0 / 1 (and its epilogue), 16 rows each, a row in four lanes: with a thread per row, four
// warps per tile, a warp had no one to share its scheduler with and issued every third cycle; 16 and 19 issue the tcgen05.mma of
// row tile 0 / 1 (an issuing thread blocks while the tensor cores are busy, and every wait or commit costs it some 90 cycles more:
// with one issuer for both tiles these were idle time of the tensor cores); 17 issues the TMA copies (queries, and keys and values
// through a ring of 128-key slots); 18 plans: it alone works out which item comes next and hands the others its bounds through
// shared memory, ahead of time (done by every warp for itself this took each some 4000 cycles per item), and it prepares the value
// tiles with masked keys.
// The CTAs stay: each takes items until none is left, so that the copies and the scores of the next item run under the epilogue
// of the one before (a CTA per item spent 7 us between the last tile of one and the first of the next).
// Every wait is bounded; on expiry the CTA records a status code, drains its copies, frees its tensor memory and returns.
#include "attn_pages.cuh"

namespace qmm {

constexpr int AT_TILE = 128;  // keys per tile, and rows per tile
constexpr int AT_SEGS = 4;  // segments planned ahead
// Up to this many sequences (two a lane) the planning warp finds its place alone, beyond the whole CTA does: 64 x 5 tokens on 200
// take 41 us, 65 x 5 take 47
constexpr int AT_FEW_SEQS = 64;
template <int HD> struct AtShape {
    static constexpr bool WIDE = HD > 128;            // one row tile, its scores in two buffers
    static constexpr int HALVES = WIDE ? 2 : 1;       // slots of a tile of keys (or values): 128 keys x up to 128 elements each
    static constexpr int NCH = (HD / HALVES + 63) / 64;  // chunks of 64 elements of a slot
    static constexpr int TILE_BYTES = NCH * AT_TILE * 128;
    static constexpr int SLOTS = NCH == 1 ? 10 : 5;   // 160 KB of keys and values
    static constexpr int ROW_TILES = WIDE ? 1 : 2, MAX_ROWS = 128 * ROW_TILES;
    // warps: softmax (eight per row tile), issuing, copying, planning, issuing for the second row tile; 20 (a 21st would leave 80 registers)
    static constexpr int SOFTMAX = 8 * ROW_TILES, MMA0 = SOFTMAX, COPY = SOFTMAX + 1, PLAN = SOFTMAX + 2, MMA1 = SOFTMAX + 3;
    static constexpr int WARPS = SOFTMAX + 2 + ROW_TILES, THREADS = 32 * WARPS;
    __host__ __device__ static constexpr uint32_t IDESC_S(bool bf16) { return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | ((AT_TILE >> 3) << 17) | ((128 >> 4) << 24); }
    __host__ __device__ static constexpr uint32_t IDESC_O(bool bf16) { return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (1u << 16) | ((HD / HALVES >> 3) << 17) | ((128 >> 4) << 24); }
};
// tensor memory columns: S of tile i at 128 i, P over the second half of S (the half that is read last goes there first), O of
// tile i at 256 + 128 i (wide heads: S of the even and odd tiles of keys at 0 and 128, O at 256)
constexpr uint32_t AT_COL_S = 0, AT_COL_P = 64, AT_COL_O = 256;

// A segment: some of the key tiles of an item, as the planning warp hands it to the others
struct AtSeg {
    int valid;          // 0: no more
    int s, q0, q_len, kv;
    int kvh, tok0, tok1;  // tokens [tok0, tok1) of the sequence
    int t0, t1;         // tiles [t0, t1) that hold keys of its rows
    int st0, st1;       // tiles of the segment before that cut
    int a, b, a2, b2;   // keys [a, b) are seen by some row, [a2, b2) by all
    int u0, u1;         // tiles [u0, u1) whose keys every row sees
    int begins, ends;   // the item's first / last segment
    int more;           // tiles of the item after the segment

    // some row does not see some key of tile t
    __device__ __forceinline__ bool masked(int t) const { return t < u0 || t >= u1; }
};

struct __align__(16) AtHeader {
    uint64_t full[10], empty[10], seg_full[AT_SEGS], seg_empty[AT_SEGS];
    AtSeg seg[AT_SEGS];
    uint64_t v_ask, v_ok, q_full, q_empty, s_full[2], p_part[2], p_full[2], o_full[2], turn[2][4], drain[2];
    long long scan[36];
    AttnParams p;  // a copy: functions that are not inlined would fetch the kernel's parameters from far away, one by one
    uint32_t tmem_base;
    int abort_flag, odd;
};
template <int HD> constexpr size_t at_smem_bytes() { return 1024 + (size_t)(2 + AtShape<HD>::SLOTS) * AtShape<HD>::TILE_BYTES + sizeof(AtHeader); }

__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc),
                 "r"(idesc), "r"(accumulate)
                 : "memory");
}
// V as the B operand, keys along K: chunks of 64 elements x 128 keys (128-byte swizzled rows); 8-key groups 1024 bytes apart, the
// next 64 elements one chunk further
__device__ __forceinline__ uint64_t umma_desc_v(uint32_t smem_addr) {
    return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)(AT_TILE * 128 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
#define QMM_R8(r, b) "=r"(r[b]), "=r"(r[b + 1]), "=r"(r[b + 2]), "=r"(r[b + 3]), "=r"(r[b + 4]), "=r"(r[b + 5]), "=r"(r[b + 6]), "=r"(r[b + 7])
#define QMM_RI8(r, b) "r"(r[b]), "r"(r[b + 1]), "r"(r[b + 2]), "r"(r[b + 3]), "r"(r[b + 4]), "r"(r[b + 5]), "r"(r[b + 6]), "r"(r[b + 7])
// Tensor memory by 16 rows (lanes 0-15 or 16-31 of the warp's quarter): lane l of the warp holds, of each block of 8 columns, columns
// 2 (l & 3) and + 1 of rows l / 4 (registers 4 i, 4 i + 1 of block i) and l / 4 + 8 (4 i + 2, 4 i + 3): a row lies in four lanes.
// The wait is part of a load: between a load and its wait nothing may touch the registers, not even a spill that the compiler
// puts there.
__device__ __forceinline__ void tmem_ld_8(uint32_t taddr, uint32_t (&r)[32]) {  // 64 columns
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : QMM_R8(r, 0), QMM_R8(r, 8), QMM_R8(r, 16), QMM_R8(r, 24)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_4(uint32_t taddr, uint32_t (&r)[16]) {  // 32 columns
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : QMM_R8(r, 0), QMM_R8(r, 8)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_4(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::QMM_RI8(r, 0),
                 QMM_RI8(r, 8), "r"(taddr)
                 : "memory");
}
// 16-bit pairs: 4 columns of 32 bits per block of 8 values; registers 2 i (row l / 4) and 2 i + 1 (row l / 4 + 8), column l & 3
__device__ __forceinline__ void tmem_st_p(uint32_t taddr, const uint32_t (&r)[16]) {  // 64 values a row: 32 columns
    asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::QMM_RI8(r, 0),
                 QMM_RI8(r, 8), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float max3(float a, float b, float c) {  // one instruction; a NaN is ignored, as by fmaxf
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}

// Scores of 64 keys from k0 on (this lane's columns of two rows): those from hi[e] on / before lo[e] do not count for row e
__device__ __forceinline__ void mask_right(uint32_t (&s)[32], int k0, const int (&hi)[2]) {
    const int n[2] = {hi[0] - k0 - 2 * ((int)threadIdx.x & 3), hi[1] - k0 - 2 * ((int)threadIdx.x & 3)};
#pragma unroll
    for (int j = 0; j < 32; ++j)
        if (8 * (j >> 2) + (j & 1) >= n[(j >> 1) & 1]) s[j] = 0xFF800000u;  // -inf
}
__device__ __forceinline__ void mask_left(uint32_t (&s)[32], int k0, const int (&lo)[2]) {
    const int n[2] = {lo[0] - k0 - 2 * ((int)threadIdx.x & 3), lo[1] - k0 - 2 * ((int)threadIdx.x & 3)};
#pragma unroll
    for (int j = 0; j < 32; ++j)
        if (8 * (j >> 2) + (j & 1) < n[(j >> 1) & 1]) s[j] = 0xFF800000u;
}
__device__ __forceinline__ void max64(const uint32_t (&s)[32], float (&m)[2]) {
#pragma unroll
    for (int j = 0; j < 32; j += 4)
#pragma unroll
        for (int e = 0; e < 2; ++e) m[e] = max3(m[e], __uint_as_float(s[j + 2 * e]), __uint_as_float(s[j + 2 * e + 1]));
}
// Two f32 operations at a time
__device__ __forceinline__ uint64_t f32x2(float a, float b) { return (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float lo2(uint64_t a) { return __uint_as_float((uint32_t)a); }
__device__ __forceinline__ float hi2(uint64_t a) { return __uint_as_float((uint32_t)(a >> 32)); }
// P = exp2((s - m) c) of 64 keys to 32 columns of tensor memory; adds this lane's columns to l (before they are rounded).  The
// difference comes first: in s c - m c, one instruction instead of two, the rounding of m c put P off by up to 2^(|m c| 2^-24), a
// factor that changed when m moved and made P overflow from |m c| = 2^28 on; the times were the same (8192 tokens within 0.5 %)
template <typename T>
__device__ __forceinline__ void exp64(const uint32_t (&s)[32], float c, const float (&mu)[2], uint32_t tp, uint64_t (&l)[2]) {
    const uint64_t c2 = f32x2(c, c);
    uint32_t pk[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const int e = j & 1;
        const uint64_t x = mul2(add2(f32x2(__uint_as_float(s[2 * j]), __uint_as_float(s[2 * j + 1])), f32x2(-mu[e], -mu[e])), c2);
        const uint64_t y = f32x2(fast_exp2(lo2(x)), fast_exp2(hi2(x)));
        l[e] = add2(l[e], y);
        pk[j] = pack2<T>(lo2(y), hi2(y));
    }
    tmem_st_p(tp, pk);
}

__device__ __forceinline__ int at_block_tokens(const AttnParams& p) { return p.row_tiles * (AT_TILE * p.group_inv >> 16); }  // of an item
__device__ __forceinline__ int at_tile_count(const KeyRange& kr) { return max(1, (max(kr.b, 0) + AT_TILE - 1) / AT_TILE - kr.a / AT_TILE); }
struct AtItems {  // items of a sequence
    __device__ static __forceinline__ int count(const AttnParams& p, int s) { return (seq_info(p, s).q_len + at_block_tokens(p) - 1) / at_block_tokens(p) * p.nkv; }
};
constexpr int AT_ITEM_COST = 2;
struct AtTiles {  // tiles of them all
    __device__ static __forceinline__ long count(const AttnParams& p, int s) {
        const SeqInfo si = seq_info(p, s);
        return (long)((si.q_len + at_block_tokens(p) - 1) / at_block_tokens(p)) * p.nkv * (at_tile_count(key_range(p, si, 0, si.q_len)) + AT_ITEM_COST);
    }
};

// The segments of this CTA, walked by the planning warp.  An item is (sequence, kv head, block of tb tokens).
// Many items: whole items, CTA c of n takes number c, 2n-1-c, 2n+c, ... of all (a sequence's last, longest blocks first, every
// second round backwards: the rounds' differences cancel).  Few items over a long axis (stream_k): all tiles are shared evenly in
// order, where every item of a sequence counts as many tiles as its last block has, at least one, and AT_ITEM_COST more (as in
// ArWalker).
struct AtWalker {
    const AttnParams& p;
    int tb;        // tokens per block
    long left;     // stream_k: places of this CTA's share still to come
    int ahead, turn;  // items from the current one to the next, rounds so far
    int s, item, within;
    SeqInfo si;
    int tl, nt, nb;

    __device__ __forceinline__ void load_seq() {
        si = seq_info(p, s);
        const KeyRange r = key_range(p, si, 0, si.q_len);
        tl = r.a / AT_TILE;
        nt = at_tile_count(r);
        nb = (si.q_len + tb - 1) / tb;
    }
    // To the item `n` after the current one; 32 sequences are looked at at a time.
    __device__ __forceinline__ bool skip(int n) {
        const int lane = threadIdx.x & 31;
        int target = item + n;
        if (target >= nb * p.nkv) {
            target -= nb * p.nkv;
#pragma unroll 1
            for (int base = s + 1;; base += 32) {
                if (base >= p.n_seqs) return false;
                const int cnt = base + lane < p.n_seqs ? AtItems::count(p, base + lane) : 0;
                int inc = cnt;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int u = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += u;
                }
                const unsigned past = __ballot_sync(0xffffffffu, inc > target);
                if (past) {
                    const int f = __ffs(past) - 1;
                    s = base + f;
                    target -= __shfl_sync(0xffffffffu, inc - cnt, f);
                    load_seq();
                    break;
                }
                target -= __shfl_sync(0xffffffffu, inc, 31);
            }
        }
        item = target;
        return true;
    }
    __device__ __forceinline__ bool next(AtSeg& g) {
        if (left <= 0) return false;
        int blk;
        if (p.stream_k) {
            while (item >= nb * p.nkv) {
                if (++s >= p.n_seqs) return false;
                item = within = 0;
                load_seq();
            }
            if (within == 0 && left <= AT_ITEM_COST) return false;  // (its first places: the item is the next CTA's)
            if (within > 0 && within <= AT_ITEM_COST) left += within, within = 0;
            const int n = (int)min(left, (long)(nt + AT_ITEM_COST - within)), w1 = within + n;
            g.kvh = item / nb, blk = item - g.kvh * nb;
            g.begins = within == 0, g.ends = w1 == nt + AT_ITEM_COST;
            g.st0 = tl + max(0, within - AT_ITEM_COST), g.st1 = tl + w1 - AT_ITEM_COST;
            left -= n, within = w1;
            g.more = nt + AT_ITEM_COST - w1;
            if (g.ends) within = 0, ++item;
        } else {
            if (!skip(ahead)) return false;
            const int n = gridDim.x, c = blockIdx.x;
            ahead = (turn++ & 1) ? 2 * c + 1 : 2 * (n - c) - 1;
            blk = item / p.nkv, g.kvh = item - blk * p.nkv, blk = nb - 1 - blk;
            g.st0 = tl, g.st1 = tl + nt;
            g.begins = g.ends = 1, g.more = 0;
        }
        g.valid = 1, g.s = s, g.q0 = si.q0, g.q_len = si.q_len, g.kv = si.kv;
        g.tok0 = blk * tb, g.tok1 = min(g.tok0 + tb, si.q_len);
        const KeyRange kr = key_range(p, si, g.tok0, g.tok1);
        g.a = kr.a, g.b = kr.b, g.a2 = kr.a2, g.b2 = kr.b2;
        g.t0 = max(g.st0, kr.a / AT_TILE), g.t1 = min(g.st1, (kr.b + AT_TILE - 1) / AT_TILE);
        g.u0 = (kr.a2 + AT_TILE - 1) / AT_TILE, g.u1 = kr.b2 / AT_TILE;
        return true;
    }
};

template <typename T, int HD>
__global__ void __launch_bounds__(AtShape<HD>::THREADS, 1) attn_tiles_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                                                                   const __grid_constant__ CUtensorMap vmap, const __grid_constant__ AttnParams params) {
    using Sh = AtShape<HD>;
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ __align__(1024) uint8_t at_raw[];
    uint8_t* sm = at_raw + ((1024u - (smem_u32(at_raw) & 1023u)) & 1023u);
    const uint32_t q_s = smem_u32(sm), ring = q_s + 2 * Sh::TILE_BYTES;
    AtHeader* hdr = reinterpret_cast<AtHeader*>(sm + (size_t)(2 + Sh::SLOTS) * Sh::TILE_BYTES);
    const AttnParams& p = hdr->p;
    volatile int* cta_abort = &hdr->abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int tpt = AT_TILE / params.group, tile_rows = tpt * params.group;  // tokens and rows of a row tile

    if (tid == 0) {
        constexpr int N = Sh::ROW_TILES;  // issuing threads
        for (int i = 0; i < Sh::SLOTS; ++i) mbar_init(smem_u32(&hdr->full[i]), 1), mbar_init(smem_u32(&hdr->empty[i]), N);
        mbar_init(smem_u32(&hdr->v_ask), N), mbar_init(smem_u32(&hdr->v_ok), 1);
        mbar_init(smem_u32(&hdr->q_full), 1), mbar_init(smem_u32(&hdr->q_empty), N);
        for (int i = 0; i < AT_SEGS; ++i) mbar_init(smem_u32(&hdr->seg_full[i]), 1), mbar_init(smem_u32(&hdr->seg_empty[i]), Sh::WARPS - 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&hdr->s_full[i]), 1), mbar_init(smem_u32(&hdr->o_full[i]), 1), mbar_init(smem_u32(&hdr->drain[i]), 1);
            mbar_init(smem_u32(&hdr->p_part[i]), 8), mbar_init(smem_u32(&hdr->p_full[i]), 8);
            for (int j = 0; j < 4; ++j) mbar_init(smem_u32(&hdr->turn[i][j]), 2);
        }
        hdr->abort_flag = 0, hdr->odd = 0;
        mbar_fence_init();
    }
    if (warp == Sh::MMA0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&hdr->tmem_base)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid < (int)(sizeof(AttnParams) / 4)) reinterpret_cast<uint32_t*>(&hdr->p)[tid] = reinterpret_cast<const uint32_t*>(&params)[tid];
    __syncthreads();
    pdl_wait_prior_grids();
    pdl_release_dependents();

    // many sequences: their lengths are read by all threads
    long total = 0, before = 0, share = 0;
    int first_seq = -1, n_ctas = 1;
    if (p.n_seqs > AT_FEW_SEQS) {
        if (p.stream_k) {
            find_item<AtTiles>(p, 1l << 62, total, hdr->scan);
            n_ctas = ar_ctas(total, gridDim.x), share = ar_share(total, min((int)blockIdx.x, n_ctas), n_ctas);
            first_seq = find_item<AtTiles>(p, share, before, hdr->scan);
        } else {
            first_seq = find_item<AtItems>(p, blockIdx.x, before, hdr->scan);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = hdr->tmem_base;

    auto wait = [&](uint64_t* bar, uint32_t phase, int code) { return wait_bar(bar, phase & 1u, code, cta_abort); };
    // The next segment (number n of this CTA) as the planning warp has laid it down, and the return of its place; whole warps
    auto have_seg = [&](int n) { return wait(&hdr->seg_full[n % AT_SEGS], n / AT_SEGS, DEV_TIMEOUT_FULL) && hdr->seg[n % AT_SEGS].valid; };
    auto done_seg = [&](int n) {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&hdr->seg_empty[n % AT_SEGS]));
    };

    if (warp == Sh::PLAN) {
        // ------------------------------------------------------------ plan: the only code that knows how items follow one another
        AtWalker w{p, Sh::ROW_TILES * tpt};
        bool any = true;
        if (p.stream_k) {
            if (p.n_seqs <= AT_FEW_SEQS) first_seq = plan_few<AtTiles>(p, total, n_ctas, share, before);
            if (lane == 0) {
                (reinterpret_cast<ArJoin*>(p.scratch) + blockIdx.x)->n_rows = 0;
                hdr->scan[34] = total, hdr->scan[35] = n_ctas;
            }
            any = (int)blockIdx.x < n_ctas && first_seq >= 0;
            if (any) {
                w.left = ar_share(total, blockIdx.x + 1, n_ctas) - share, w.s = first_seq;
                w.load_seq();
                const long ahead = share - before;
                w.item = (int)(ahead / (w.nt + AT_ITEM_COST)), w.within = (int)(ahead - (long)w.item * (w.nt + AT_ITEM_COST));
            }
        } else {
            w.s = first_seq, w.item = w.nb = w.within = 0, w.left = 1, w.ahead = blockIdx.x, w.turn = 0;
            if (p.n_seqs > AT_FEW_SEQS) {
                any = first_seq >= 0;
                if (any) {
                    w.load_seq();
                    w.item = (int)(blockIdx.x - before), w.ahead = 0;
                }
            }
        }
        // It also prepares the value tiles with keys that some row does not see (clear_values: the tensor cores add 0 * v there),
        // those of a segment after the next one is laid down.  The issuers ask for each such tile when it has landed and wait for
        // it before they ask for the next: this warp does not follow the ring's own barriers, most of whose phases it would skip.
        if (!any) {  // nothing to do for this CTA
            if (lane == 0) {
                hdr->seg[0].valid = 0;
                mbar_arrive(smem_u32(&hdr->seg_full[0]));
            }
            __syncwarp();
        }
        int it = 0;
        uint32_t n_v = 0;
        AtSeg last = {};
        bool ok = true;
        for (int n = 0; ok && any; ++n) {
            AtSeg g = {};
            any = any && w.next(g);
            if (n >= AT_SEGS && !wait(&hdr->seg_empty[n % AT_SEGS], n / AT_SEGS - 1, DEV_TIMEOUT_EMPTY)) break;
            if (lane == 0) {
                hdr->seg[n % AT_SEGS] = g;
                mbar_arrive(smem_u32(&hdr->seg_full[n % AT_SEGS]));
            }
            __syncwarp();
            const int tiles = max(last.t1 - last.t0, 0);
            for (int k = 0; k < tiles; ++k) {
                const int t = last.t0 + k;
                if (!last.masked(t)) continue;
                if (!wait(&hdr->v_ask, n_v++, DEV_TIMEOUT_FULL)) {
                    ok = false;
                    break;
                }
                const int k0 = t * AT_TILE, left = min(max(last.a2 - k0, 0), AT_TILE), right = min(max(last.b2 - k0, left), AT_TILE);
                bool odd = false;
                // order of the slots: K0 V0 K1 V1 ..., or (scores one tile ahead) K0 K1 V0 K2 V1 ...
                const int v_it = it + (Sh::WIDE ? 2 * (min(k + 2, tiles) + k) : 2 * k + 1);
#pragma unroll 1
                for (int ch = 0; ch < Sh::NCH * Sh::HALVES; ++ch) {
                    uint4* vp = reinterpret_cast<uint4*>(sm + (size_t)(2 + (v_it + ch / Sh::NCH) % Sh::SLOTS) * Sh::TILE_BYTES) + (ch % Sh::NCH) * AT_TILE * 8;
                    if (left > 0) odd |= clear_values<T, 8>(vp, 0, left, last.a - k0, last.b - k0, lane, 32);
                    odd |= clear_values<T, 8>(vp, right, AT_TILE, last.a - k0, last.b - k0, lane, 32);
                }
                if (odd) *reinterpret_cast<volatile int*>(&hdr->odd) = 1;  // (stays set: the rows of later segments are looked at too)
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // read by the tensor cores, refilled by a copy
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&hdr->v_ok));
            }
            it += 2 * Sh::HALVES * tiles;
            last = g;
        }
    } else if (warp == Sh::COPY) {
        // ------------------------------------------------------------ copies
        int it = 0, q_no = 0;  // tiles (of keys and of values) and query blocks so far
        bool ok = true;
        for (int n = 0; ok && have_seg(n); done_seg(n), ++n) {
            const AtSeg& w = hdr->seg[n % AT_SEGS];
            const int t0 = w.t0, t1 = w.t1, kvh = w.kvh, q0 = w.q0;
            if (t0 >= t1) continue;
            const int nq = Sh::WIDE || w.tok1 - w.tok0 > tpt ? 2 : 1;
            int first, cnt, pages, slots;
            tile_boxes<AT_TILE>(p, t0, w.a, w.b, first, cnt);
            pages = page_of_boxes<AT_TILE>(p, w.s, q0, t0, first, cnt, slots);
            if (q_no > 0 && !wait(&hdr->q_empty, q_no - 1, DEV_TIMEOUT_EMPTY)) break;
            if (lane == 0) mbar_arrive_expect_tx(smem_u32(&hdr->q_full), (uint32_t)(nq * Sh::NCH * tile_rows * 128));
            __syncwarp();
            if (lane < nq * Sh::NCH) {  // (nq: row tiles, or halves of the elements)
                const int i = lane / Sh::NCH, c = lane % Sh::NCH;
                tma_load_3d(q_s + (uint32_t)(i * Sh::TILE_BYTES + c * AT_TILE * 128), &qmap, (Sh::WIDE ? lane : c) * 64, kvh * p.group,
                            q0 + w.tok0 + (Sh::WIDE ? 0 : i * tpt), smem_u32(&hdr->q_full));
            }
            ++q_no;
            auto load = [&](const CUtensorMap* map, int t, int first, int cnt, int pages, int slots) {
#pragma unroll 1
                for (int h = 0; h < Sh::HALVES; ++h, ++it) {
                    const int sl = it % Sh::SLOTS;
                    if (it >= Sh::SLOTS && !wait(&hdr->empty[sl], it / Sh::SLOTS - 1, DEV_TIMEOUT_EMPTY)) return false;
                    const uint32_t bar = smem_u32(&hdr->full[sl]);
                    if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(cnt * Sh::NCH * 128) << p.box_shift);
                    __syncwarp();
                    load_tile<AT_TILE, Sh::NCH>(p, map, ring + (uint32_t)sl * Sh::TILE_BYTES, bar, h * 128, first, cnt, pages, slots, kvh);
                }
                return true;
            };
            for (int t = t0; t < t1 && ok; ++t) {
                int nfirst = 0, ncnt = 0, npages = 0, nslots = 0;
                if (t + 1 < t1) {  // the next tile's pages are looked up before its turn comes
                    tile_boxes<AT_TILE>(p, t + 1, w.a, w.b, nfirst, ncnt);
                    npages = page_of_boxes<AT_TILE>(p, w.s, q0, t + 1, nfirst, ncnt, nslots);
                }
                if (Sh::WIDE) {
                    if (t == t0) ok = load(&kmap, t, first, cnt, pages, slots);
                    if (ok && t + 1 < t1) ok = load(&kmap, t + 1, nfirst, ncnt, npages, nslots);
                } else {
                    ok = load(&kmap, t, first, cnt, pages, slots);
                }
                ok = ok && load(&vmap, t, first, cnt, pages, slots);
                first = nfirst, cnt = ncnt, pages = npages, slots = nslots;
            }
        }
        if (*cta_abort) {  // copies in flight land before the CTA ends
#pragma unroll 1
            for (int i = max(0, it - Sh::SLOTS); i <= it; ++i) {
                uint64_t* bar = i < it ? &hdr->full[i % Sh::SLOTS] : &hdr->q_full;
                const uint32_t ph = i < it ? (i / Sh::SLOTS) & 1 : (q_no - 1) & 1;
                if (i == it && q_no == 0) break;
                const long long c0 = clock64();
                while (!mbar_try_wait(smem_u32(bar), ph))
                    if (clock64() - c0 > WAIT_LIMIT_CYCLES) {
                        raise_status(DEV_TIMEOUT_DRAIN);
                        break;
                    }
            }
        }
    } else if (Sh::WIDE && warp == Sh::MMA0) {
        // ------------------------------------------------------------ tensor cores, wide heads: scores one tile ahead of the outputs
        // (one row tile, so its scores have two buffers and the next ones are ready when a softmax ends)
        int it = 0, q_no = 0;
        uint32_t j = 0, n_v = 0;  // tiles so far (their scores are in buffer j & 1), value tiles handed to the planning warp
        bool ok = true;
        const uint64_t qd = umma_desc_sw128(q_s);
        auto release = [&](uint64_t* bar) {
            if (lane == 0) umma_commit(smem_u32(bar));
        };
        auto scores = [&](uint32_t jj) {
            for (int h = 0; h < Sh::HALVES; ++h, ++it) {
                const int sl = it % Sh::SLOTS;
                if (!wait(&hdr->full[sl], it / Sh::SLOTS, DEV_TIMEOUT_FULL)) return false;
                tc_fence_after();
                if (lane == 0) {
                    const uint64_t kd = umma_desc_sw128(ring + (uint32_t)sl * Sh::TILE_BYTES), qh = qd + (uint64_t)(h * (Sh::TILE_BYTES >> 4));
#pragma unroll
                    for (int k16 = 0; k16 < 8; ++k16) {
                        const uint64_t off = (uint64_t)((k16 >> 2) * (AT_TILE * 128 >> 4) + (k16 & 3) * 2);
                        umma_bf16(tmem + AT_COL_S + 128u * (jj & 1), qh + off, kd + off, Sh::IDESC_S(BF16), h > 0 || k16 > 0);
                    }
                }
                release(&hdr->empty[sl]);
            }
            release(&hdr->s_full[jj & 1]);
            return true;
        };
        for (int n = 0; ok && have_seg(n); done_seg(n), ++n) {
            const AtSeg& w = hdr->seg[n % AT_SEGS];
            const int t0 = w.t0, t1 = w.t1, u0 = w.u0, u1 = w.u1;
            if (t0 >= t1) continue;
            if (!wait(&hdr->q_full, q_no, DEV_TIMEOUT_FULL)) break;
            ++q_no;
            ok = scores(j) && (t0 + 1 >= t1 || scores(j + 1));
            if (ok && t0 + 2 >= t1) release(&hdr->q_empty);
            for (int t = t0; t < t1 && ok; ++t, ++j) {
                const int s0 = it % Sh::SLOTS, s1 = (it + 1) % Sh::SLOTS;
                ok = wait(&hdr->full[s0], it / Sh::SLOTS, DEV_TIMEOUT_FULL) && wait(&hdr->full[s1], (it + 1) / Sh::SLOTS, DEV_TIMEOUT_FULL);
                if (ok && (t < u0 || t >= u1)) {  // keys that some row does not see: prepared by the planning warp
                    if (lane == 0) mbar_arrive(smem_u32(&hdr->v_ask));
                    ok = wait(&hdr->v_ok, n_v++, DEV_TIMEOUT_FULL);
                }
                for (int part = 1; part >= 0 && ok; --part) {  // the second half of the keys first, as its probabilities come
                    ok = wait(part ? &hdr->p_part[0] : &hdr->p_full[0], j, DEV_TIMEOUT_MMA);
                    if (!ok) break;
                    tc_fence_after();
                    if (lane == 0) {
                        const uint64_t v0 = umma_desc_v(ring + (uint32_t)s0 * Sh::TILE_BYTES), v1 = umma_desc_v(ring + (uint32_t)s1 * Sh::TILE_BYTES);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t pt = tmem + AT_COL_S + 128u * (j & 1) + AT_COL_P + 8u * (4 * part + k), acc = t > t0 || part == 0 || k > 0;
                            umma_ts(tmem + AT_COL_O, pt, v0 + (uint64_t)((4 * part + k) * (2048 >> 4)), Sh::IDESC_O(BF16), acc);
                            umma_ts(tmem + AT_COL_O + 128u, pt, v1 + (uint64_t)((4 * part + k) * (2048 >> 4)), Sh::IDESC_O(BF16), acc);
                        }
                    }
                }
                if (!ok) break;
                release(&hdr->o_full[0]);
                release(&hdr->empty[s0]);
                release(&hdr->empty[s1]);
                it += 2;
                if (t + 2 < t1) {
                    ok = scores(j + 2);
                    if (t + 3 >= t1) release(&hdr->q_empty);
                }
            }
        }
        __syncwarp();
        if (*cta_abort) {  // what was issued retires before the tensor memory is freed
            if (lane == 0) {
                umma_commit(smem_u32(&hdr->drain[0]));
                const long long c0 = clock64();
                while (!mbar_try_wait(smem_u32(&hdr->drain[0]), 0))
                    if (clock64() - c0 > WAIT_LIMIT_CYCLES) {
                        raise_status(DEV_TIMEOUT_DRAIN);
                        break;
                    }
            }
            __syncwarp();
        }
    } else if (!Sh::WIDE && (warp == Sh::MMA0 || warp == Sh::MMA1)) {
        // ------------------------------------------------------------ tensor cores: row tile i (one thread issues)
        // Both issuers follow every segment and every slot, also where there is no second row tile: a barrier whose phases one of
        // them skipped could not be waited for by parity.
        const int i = warp == Sh::MMA0 ? 0 : 1;
        const uint32_t d_s = tmem + AT_COL_S + 128u * i, d_o = tmem + AT_COL_O + 128u * i;
        const uint64_t qd = umma_desc_sw128(q_s + (uint32_t)i * Sh::TILE_BYTES);
        int it = 0, q_no = 0;
        uint32_t n_p = 0, n_v = 0;  // P tiles awaited, value tiles handed to the planning warp so far
        bool ok = true, active = false;
        auto mma_s = [&](int slot) {
            const uint64_t kd = umma_desc_sw128(ring + (uint32_t)slot * Sh::TILE_BYTES);
#pragma unroll
            for (int k16 = 0; k16 < HD / 16; ++k16) {  // 32 bytes of a 128-byte row each; the next 64 elements one chunk further
                const uint64_t off = (uint64_t)((k16 >> 2) * (AT_TILE * 128 >> 4) + (k16 & 3) * 2);
                umma_bf16(d_s, qd + off, kd + off, Sh::IDESC_S(BF16), k16 > 0);
            }
            umma_commit(smem_u32(&hdr->s_full[i]));
        };
        auto mma_o = [&](int slot, int first, int last, bool acc) {  // 16 keys each: 8 columns of P, 2048 bytes of V
            const uint64_t vd = umma_desc_v(ring + (uint32_t)slot * Sh::TILE_BYTES);
#pragma unroll
            for (int k16 = first; k16 < last; ++k16)
                umma_ts(d_o, d_s + AT_COL_P + 8u * k16, vd + (uint64_t)(k16 * (2048 >> 4)), Sh::IDESC_O(BF16), (acc || k16 > first) ? 1u : 0u);
        };
        auto release = [&](uint64_t* bar) {  // when what this thread has issued so far retires
            if (lane == 0) {
                if (active) umma_commit(smem_u32(bar));
                else mbar_arrive(smem_u32(bar));
            }
        };
        // a value tile with keys that some row does not see goes through the planning warp while its scores are in softmax
        auto ask_v = [&](bool masked, int v_it) {
            if (!masked) return true;
            if (!wait(&hdr->full[v_it % Sh::SLOTS], v_it / Sh::SLOTS, DEV_TIMEOUT_FULL)) return false;
            if (lane == 0) mbar_arrive(smem_u32(&hdr->v_ask));
            ++n_v;
            return true;
        };
        for (int n = 0; ok && have_seg(n); done_seg(n), ++n) {
            const AtSeg& w = hdr->seg[n % AT_SEGS];
            const int t0 = w.t0, t1 = w.t1, u0 = w.u0, u1 = w.u1;
            if (t0 >= t1) continue;
            active = i == 0 || w.tok1 - w.tok0 > tpt;
            int sl = it % Sh::SLOTS;
            if (!wait(&hdr->q_full, q_no, DEV_TIMEOUT_FULL) || !wait(&hdr->full[sl], it / Sh::SLOTS, DEV_TIMEOUT_FULL)) break;
            ++q_no;
            tc_fence_after();
            if (active && lane == 0) mma_s(sl);
            release(&hdr->empty[sl]);
            if (t0 + 1 == t1) release(&hdr->q_empty);
            ++it;
            ok = ask_v(t0 < u0 || t0 >= u1, it);
            for (int t = t0; t < t1 && ok; ++t) {
                const int vs = it % Sh::SLOTS, ks = (it + 1) % Sh::SLOTS;
                const bool more = t + 1 < t1;
                ok = wait(&hdr->full[vs], it / Sh::SLOTS, DEV_TIMEOUT_FULL);
                if (ok && (t < u0 || t >= u1)) ok = wait(&hdr->v_ok, n_v - 1, DEV_TIMEOUT_FULL);
                if (ok && more) ok = wait(&hdr->full[ks], (it + 1) / Sh::SLOTS, DEV_TIMEOUT_FULL);
                if (ok && active) {
                    ok = wait(&hdr->p_part[i], n_p, DEV_TIMEOUT_MMA);
                    if (!ok) break;
                    tc_fence_after();
                    if (lane == 0) mma_o(vs, 4, 8, t > t0);
                    ok = wait(&hdr->p_full[i], n_p, DEV_TIMEOUT_MMA);
                    if (!ok) break;
                    ++n_p;
                    tc_fence_after();
                    if (lane == 0) {
                        mma_o(vs, 0, 4, true);
                        if (more) mma_s(ks);
                        else umma_commit(smem_u32(&hdr->o_full[i]));
                    }
                }
                if (!ok) break;
                release(&hdr->empty[vs]);
                if (more) {
                    release(&hdr->empty[ks]);
                    if (t + 2 == t1) release(&hdr->q_empty);
                }
                it += more ? 2 : 1;
                if (more) ok = ask_v(t + 1 < u0 || t + 1 >= u1, it);
            }
        }
        __syncwarp();
        if (*cta_abort) {  // what was issued retires before the tensor memory is freed
            if (lane == 0) {
                umma_commit(smem_u32(&hdr->drain[i]));
                const long long c0 = clock64();
                while (!mbar_try_wait(smem_u32(&hdr->drain[i]), 0))
                    if (clock64() - c0 > WAIT_LIMIT_CYCLES) {
                        raise_status(DEV_TIMEOUT_DRAIN);
                        break;
                    }
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------------------ softmax and epilogue: 16 rows per warp
        const int wg = warp >> 3, row0 = (warp & 3) * 32 + ((warp >> 2) & 1) * 16 + (lane >> 2);  // this lane's rows: row0, row0 + 8
        const uint32_t lanes = (uint32_t)((warp & 3) * 32 + ((warp >> 2) & 1) * 16) << 16;
        uint32_t ts = tmem + lanes + AT_COL_S + 128u * wg;
        const uint32_t to = tmem + lanes + AT_COL_O + 128u * wg;
        uint32_t n_s = 0, n_o = 0, n_turn = 0;
        const float c = p.scale_log2;
        bool ok = true;
        for (int n = 0; ok && have_seg(n); done_seg(n), ++n) {
            const AtSeg& w = hdr->seg[n % AT_SEGS];
            const int t0 = w.t0, t1 = w.t1, u0 = w.u0, u1 = w.u1, pos0 = w.kv - w.q_len;
            const int n_tok = w.tok1 - w.tok0;
            const bool both = !Sh::WIDE && n_tok > tpt;
            if (wg == 1 && !both) continue;  // no rows in this row tile
            int lo[2], hi[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int tok = w.tok0 + wg * tpt + ((row0 + 8 * e) * p.group_inv >> 16), pos = pos0 + tok;
                hi[e] = row0 + 8 * e < tile_rows && tok < w.tok1 ? max(pos + 1, 0) : 0;
                lo[e] = first_key(p, pos);
            }
            float m[2] = {-INFINITY, -INFINITY};
            uint64_t l2[2] = {0ull, 0ull};  // sums of this lane's even and odd columns
            for (int t = t0; t < t1; ++t) {
                if (Sh::WIDE) ts = tmem + lanes + AT_COL_S + 128u * (n_s & 1);
                if (!wait(Sh::WIDE ? &hdr->s_full[n_s & 1] : &hdr->s_full[wg], Sh::WIDE ? n_s >> 1 : n_s, DEV_TIMEOUT_MMA)) {
                    ok = false;
                    break;
                }
                ++n_s;
                tc_fence_after();
                // The rows' maxima from both halves of the keys; the second half stays in registers, the first is read again for
                // its exponentials
                const bool right = t >= u1, left = t < u0;
                uint32_t sr[32];
                float mt[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                    tmem_ld_8(ts + 64 * h, sr);
                    if (right) mask_right(sr, t * AT_TILE + 64 * h, hi);
                    if (left) mask_left(sr, t * AT_TILE + 64 * h, lo);
                    max64(sr, mt);
                }
                bool grew = false;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    mt[e] = fmaxf(mt[e], __shfl_xor_sync(0xffffffffu, mt[e], 1));
                    mt[e] = fmaxf(mt[e], __shfl_xor_sync(0xffffffffu, mt[e], 2));
                    // A row's maximum moves by what the row itself has seen, not when another row of the warp makes it rescale: the
                    // roundings of P depend on it.  (Rows that are none, hi 0, hold anything: reruns would not be bit identical)
                    if (t == t0 || (hi[e] > 0 && ((mt[e] - m[e]) * c > 8.f || (m[e] == -INFINITY && mt[e] > -INFINITY)))) grew = true;
                    else mt[e] = m[e];
                }
                bool o_done = !Sh::WIDE || t == t0;  // the outputs so far are complete (two row tiles: they are when the scores are)
                if (t == t0) {
                    m[0] = mt[0], m[1] = mt[1];
                } else if (__any_sync(0xffffffffu, grew)) {
                    if (!o_done) {
                        if (!wait(&hdr->o_full[0], n_o, DEV_TIMEOUT_MMA)) {
                            ok = false;
                            break;
                        }
                        ++n_o, o_done = true;
                        tc_fence_after();
                    }
                    float f[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        f[e] = mt[e] == m[e] ? 1.f : fast_exp2((m[e] - mt[e]) * c);
                        m[e] = mt[e], l2[e] = mul2(l2[e], f32x2(f[e], f[e]));
                    }
#pragma unroll 1
                    for (int q = 0; q < HD / 32; ++q) {
                        uint32_t r[16];
                        tmem_ld_4(to + 32 * q, r);
#pragma unroll
                        for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * f[(j >> 1) & 1]);
                        tmem_st_4(to + 32 * q, r);
                    }
                }
                // The two row tiles take turns at the exponentials: left to themselves both wait for scores at the same time and then
                // share the special-function units, while the tensor cores idle (8192 tokens, 32/8 heads, when the turns were added:
                // 619 us without, 550 with; handed over after half of the keys: 633; a quarter of the exponentials as polynomials
                // instead: slower, the schedulers' issue slots bound it then).  Per scheduler, warp & 3: whoever is ready there goes on
                if (both) {
                    if ((wg == 1 || n_turn > 0) && !wait(&hdr->turn[wg][warp & 3], wg == 1 ? n_turn : n_turn - 1, DEV_TIMEOUT_MMA)) {
                        ok = false;
                        break;
                    }
                    ++n_turn;
                }
                const float mu[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll 1
                for (int h = 1; h >= 0; --h) {  // the second half, in registers, first
                    if (h == 0) {
                        tmem_ld_8(ts, sr);
                        if (right) mask_right(sr, t * AT_TILE, hi);
                        if (left) mask_left(sr, t * AT_TILE, lo);
                    }
                    exp64<T>(sr, c, mu, ts + AT_COL_P + 32 * h, l2);
                    if (h == 1 && !o_done) {  // once per tile, and before P is announced: the issuer is then past the P before
                        ok = wait(&hdr->o_full[0], n_o, DEV_TIMEOUT_MMA);
                        ++n_o;
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(h ? &hdr->p_part[wg] : &hdr->p_full[wg]));  // the product of this half can begin
                }
                if (!ok) break;
                if (both && lane == 0) mbar_arrive(smem_u32(&hdr->turn[wg ^ 1][warp & 3]));
            }
            if (!ok) break;
            if (t0 < t1) {
                if (!wait(&hdr->o_full[wg], n_o, DEV_TIMEOUT_MMA)) break;
                ++n_o;
                tc_fence_after();
            }
            const bool whole = w.begins && w.ends;
            const int slot = 2 * (int)blockIdx.x + (w.begins ? 1 : 0);
            float* ml = whole ? nullptr : ArScratch<HD, Sh::MAX_ROWS>::ml(p.scratch, gridDim.x, slot);
            float* so = whole ? nullptr : ArScratch<HD, Sh::MAX_ROWS>::o(p.scratch, gridDim.x, slot);
            {
                // each lane its own columns, 8 or 4 bytes a time (turning them within the four lanes of a row for wider stores took
                // three times the instructions, which are what bounds this part)
                char* dst[2];
                uint64_t inv[2];
                bool live[2];
                const bool f32 = !whole || p.out_dtype == QMM_DT_F32, f16 = p.out_dtype == QMM_DT_F16;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = row0 + 8 * e, tk = row * p.group_inv >> 16, g = row - tk * p.group, tok = w.tok0 + wg * tpt + tk;
                    float l = lo2(l2[e]) + hi2(l2[e]);
                    l += __shfl_xor_sync(0xffffffffu, l, 1);
                    l += __shfl_xor_sync(0xffffffffu, l, 2);
                    live[e] = row < tile_rows && tok < w.tok1;
                    const float i = !whole ? 1.f : pos0 + tok >= 0 ? 1.f / l : 0.f;  // (a row that sees no key has zeros)
                    inv[e] = f32x2(i, i);
                    const int r = (tok - w.tok0) * p.group + g;  // row of the item
                    const size_t oe = (size_t)(w.q0 + tok) * p.out_stride + (size_t)(w.kvh * p.group + g) * HD;
                    dst[e] = (whole ? static_cast<char*>(p.out) + oe * (f32 ? 4 : 2) : reinterpret_cast<char*>(so + (size_t)r * HD)) + (lane & 3) * (f32 ? 8 : 4);
                    if (!whole && live[e] && (lane & 3) == 0) ml[2 * r] = m[e], ml[2 * r + 1] = l;
                }
#pragma unroll 2
                for (int q = 0; q < HD / 32; ++q) {
                    uint32_t o[16];
                    if (t0 < t1) {
                        tmem_ld_4(to + 32 * q, o);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] = 0u;
                    }
                    uint64_t v[8];  // block i of 8 columns, row e: v[2 i + e]
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint64_t x = f32x2(__uint_as_float(o[2 * j]), __uint_as_float(o[2 * j + 1]));
                        v[j] = mul2(x, inv[j & 1]);
                    }
                    if (f32) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (live[j & 1]) *reinterpret_cast<float2*>(dst[j & 1] + (32 * q + 8 * (j >> 1)) * 4) = make_float2(lo2(v[j]), hi2(v[j]));
                    } else {
                        uint32_t h[8];
                        if (f16) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) h[j] = pack2<__half>(lo2(v[j]), hi2(v[j]));
                        } else {
#pragma unroll
                            for (int j = 0; j < 8; ++j) h[j] = pack2<__nv_bfloat16>(lo2(v[j]), hi2(v[j]));
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (live[j & 1]) *reinterpret_cast<uint32_t*>(dst[j & 1] + (32 * q + 8 * (j >> 1)) * 2) = h[j];
                    }
                }
                if (*reinterpret_cast<volatile int*>(&hdr->odd)) {
                    const int lo_k = max(w.a, w.st0 * AT_TILE), hi_k = min(w.b, w.st1 * AT_TILE), left = min(max(w.a2, lo_k), hi_k), right = max(min(w.b2, hi_k), left);
                    // the warp's rows of the item
                    const int base = w.tok0 * p.group, first = wg * tile_rows + row0 - (lane >> 2), end = min(min(first + 16, (wg + 1) * tile_rows), n_tok * p.group);
                    add_odd_values<T, HD>(p, w.s, w.q0, pos0, w.kvh, lo_k, left, base + first, base + end, so, base);
                    add_odd_values<T, HD>(p, w.s, w.q0, pos0, w.kvh, right, hi_k, base + first, base + end, so, base);
                }
            }
            if (w.begins && !w.ends && tid == 0) {  // this item goes on in the next CTAs: how many of them
                ArJoin j;
                j.s = w.s, j.q0 = w.q0, j.tok_row0 = w.tok0 * p.group, j.n_rows = n_tok * p.group, j.kvh = w.kvh;
                j.any_key = pos0;
                const long total = hdr->scan[34];
                const int n_ctas = (int)hdr->scan[35];
                const long item_end = ar_share(total, blockIdx.x + 1, n_ctas) + w.more;  // (a segment that does not end its item ends the share)
                j.n_parts = ar_last(total, item_end, n_ctas) - (int)blockIdx.x + 1, j.pad = 0;
                reinterpret_cast<ArJoin*>(p.scratch)[blockIdx.x] = j;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == Sh::MMA0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---- host side ----
template <typename T, int HD>
static int attn_tiles_inst(const AttnParams& p, const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s) {
    constexpr size_t smem = at_smem_bytes<HD>();
    static std::mutex mu;
    static bool configured[64] = {};
    int dev = 0;
    QMM_CUDA_TRY(cudaGetDevice(&dev));
    {
        std::lock_guard<std::mutex> g(mu);
        if (dev < 0 || dev >= 64 || !configured[dev]) {
            QMM_CUDA_TRY(cudaFuncSetAttribute(attn_tiles_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            if (dev >= 0 && dev < 64) configured[dev] = true;
        }
    }
    const int tb = AtShape<HD>::ROW_TILES * (AT_TILE / p.group), ctas = sm_count();
    const long items = ((long)p.total_q / tb + p.n_seqs) * p.nkv;  // at least as many as there are
    if (items > 1l << 30) return QMM_ERR_UNSUPPORTED;
    const int grid = p.stream_k ? ctas : (int)(items < ctas ? items : ctas);
    if (int st = launch_overlapped(attn_tiles_kernel<T, HD>, dim3(grid), dim3(AtShape<HD>::THREADS), smem, s, qm, km, vm, p)) return st;
    if (p.stream_k) return launch_overlapped(attn_join_kernel<HD, AtShape<HD>::MAX_ROWS>, dim3(ctas, AtShape<HD>::MAX_ROWS / 4), dim3(128), 0, s, p, ctas);
    return QMM_OK;
}
template <int HD> static long at_scratch_bytes_of() { return 4 * (long)ArScratch<HD, AtShape<HD>::MAX_ROWS>::floats(sm_count()); }
static long attn_tiles_scratch_bytes(int hd) {
    switch (hd) {
    case 32: return at_scratch_bytes_of<32>();
    case 64: return at_scratch_bytes_of<64>();
    case 96: return at_scratch_bytes_of<96>();
    case 128: return at_scratch_bytes_of<128>();
    case 256: return at_scratch_bytes_of<256>();
    }
    return QMM_ERR_UNSUPPORTED;
}
// The queries as (element, head, row), a box = the rows of one row tile: tokens outermost, the heads of a group inside
static int attn_tiles_rows(int hd) { return hd <= 128 ? 256 : 128; }  // of an item
static int attn_tiles_launch(const AttnParams& p, const CUtensorMap& km, const CUtensorMap& vm, int dtype, int hd, cudaStream_t s) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return cuda_fail(cudaErrorNotSupported);
    CUtensorMap qm;
    const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)p.nqh, (cuuint64_t)p.total_q};
    const cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)p.q_stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)p.group, (cuuint32_t)(AT_TILE / p.group)}, estr[3] = {1, 1, 1};
    if (enc(&qm, dtype == QMM_DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p.q), dims, strides, box,
            estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cuda_fail(cudaErrorInvalidValue);
    const bool f16 = dtype == QMM_DT_F16;
    switch (hd) {
    case 32: return f16 ? attn_tiles_inst<__half, 32>(p, qm, km, vm, s) : attn_tiles_inst<__nv_bfloat16, 32>(p, qm, km, vm, s);
    case 64: return f16 ? attn_tiles_inst<__half, 64>(p, qm, km, vm, s) : attn_tiles_inst<__nv_bfloat16, 64>(p, qm, km, vm, s);
    case 96: return f16 ? attn_tiles_inst<__half, 96>(p, qm, km, vm, s) : attn_tiles_inst<__nv_bfloat16, 96>(p, qm, km, vm, s);
    case 128: return f16 ? attn_tiles_inst<__half, 128>(p, qm, km, vm, s) : attn_tiles_inst<__nv_bfloat16, 128>(p, qm, km, vm, s);
    case 256: return f16 ? attn_tiles_inst<__half, 256>(p, qm, km, vm, s) : attn_tiles_inst<__nv_bfloat16, 256>(p, qm, km, vm, s);
    }
    return QMM_ERR_UNSUPPORTED;
}

}  // namespace qmm
