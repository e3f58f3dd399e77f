// Attention of one or a few new tokens per sequence over a paged cache (decode) on mma.sync.  The counterpart, for a batch of
// sequences of different lengths, of the upstream's gpu_gqa_attn_into (gpu-core/src/infer_ops.rs:160-189).
//
//   out[r, h] = sum_t w_t V_t / sum_t w_t,  w_t = exp(kq_scale * q_r . K_t - max),  t in (pos_r - window, pos_r]
//
// One pass over the keys with a running maximum and sum.  The rows of a work item (up to 16) are (token, query head of the group)
// pairs of ONE kv head, so a tile of keys and values fetched once serves every query head that shares it.  Bound by the cache bytes:
// the four math warps take 16 keys each of a tile of 64 and join at the end; a fifth warp plans and keeps TMA copies of the next
// tiles in flight.
// Few items over a long axis: all (item, tile) pairs are shared out evenly over the CTAs, whatever the sequences' lengths
// (read on the device: nothing is copied to the host).  A CTA's share begins and ends inside at most two items; those go to
// scratch as (maximum, sum, unnormalised output) and attn_join_kernel adds them in key order, so reruns are bit identical.
// q, k, v are f16 or bf16; the probabilities are rounded to the same type for the second product (tensor-core operands),
// scores, maximum, sum and output stay f32.
// Measured: 64 sequences of 91 to 8192 keys, 64/8 heads of 128, bf16: 106 us, 5.3 TB/s of cache; one sequence of 131001 keys,
// 32/8 heads: 93 us, 5.8 TB/s; one of 2048: 12.5 us, of which the first copy is under way after 4 and the joining takes 3.
#include "attn_pages.cuh"

namespace qmm {

constexpr int AR_TILE = 64;       // keys per tile
constexpr int AR_ROWS = 16;       // rows of an item
constexpr int AR_THREADS = 160;   // four math warps and the copying warp
template <int HD> struct ArShape {
    static constexpr int NCH = (HD + 63) / 64;
    static constexpr int TILE_BYTES = NCH * AR_TILE * 128;  // one matrix
    // two CTAs per SM up to 128 elements, about 96 KB of tiles each (bytes in flight); one with 192 KB at 256
    static constexpr int STAGES = HD <= 64 ? 6 : 3;
    static constexpr int CTAS_PER_SM = HD <= 128 ? 2 : 1;
    static constexpr int BUF_PITCH = HD + 4;
    static constexpr bool Q_REGS = HD <= 128;  // the queries stay in registers (wider heads read them from shared memory)
};

constexpr int AR_SEGS = 4;  // segments planned ahead
constexpr int AR_FEW_SEQS = 64;  // up to this many sequences the copying warp plans alone (64 decodes on 200 take 22.8 us, 65 take 23.4)
// A segment: some of the key tiles of an item, as the copying warp hands it to the math warps
struct ArSeg {
    int valid;            // 0: no more
    int s, q0, q_len, kv, kvh;
    int r0, n_rows;       // rows r0 .. + n_rows of the sequence's (token, head of the group) list
    int t0, t1;           // tiles [t0, t1) that hold keys of the rows
    int st0, st1;         // tiles of the segment before that cut
    int a, b, a2, b2;     // keys [a, b) are seen by some row, [a2, b2) by all
    int begins, ends;     // the item's first / last segment
    int more;             // tiles of the item after the segment
};

struct __align__(16) ArHeader {
    uint64_t full[8], empty[8], seg_full[AR_SEGS], seg_empty[AR_SEGS], q_full, q_empty;
    ArSeg seg[AR_SEGS];
    long long scan[36];
    float ml[4][16][2];
    AttnParams p;  // a copy: functions that are not inlined would fetch the kernel's parameters from far away, one by one
    int abort_flag, odd;
};

template <int HD> constexpr size_t ar_smem_bytes() {
    using Sh = ArShape<HD>;
    return 1024 + (size_t)Sh::STAGES * 2 * Sh::TILE_BYTES + (size_t)AR_ROWS * (Sh::NCH * 64 + 8) * 2 + AR_ROWS * Sh::BUF_PITCH * 4 + sizeof(ArHeader);
}

// What a CTA leaves in scratch for attn_join_kernel: the item that begins in it and continues in later CTAs
struct ArJoin {
    int s, q0, tok_row0, n_rows;  // rows tok_row0 .. + n_rows of the sequence's (token, head of the group) list; n_rows 0: none
    int kvh, n_parts, any_key, pad;
};

template <typename T>
__device__ __forceinline__ void mma_16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    mma_f16_k16(d, a0, a1, a2, a3, b0, b1);
}
template <>
__device__ __forceinline__ void mma_16<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void math_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

__device__ __forceinline__ int ar_tile_count(const KeyRange& kr) { return max(1, (max(kr.b, 0) + AR_TILE - 1) / AR_TILE - kr.a / AR_TILE); }
constexpr int AR_ITEM_COST = 2;

// Walks the segments (item, tiles of it) of this CTA (the copying warp).  An item is (sequence, kv head, block of AR_ROWS rows); all items
// of a sequence count the tiles of the whole sequence, at least one, and AR_ITEM_COST more for what an item costs beside its tiles
// (its queries, the joining of its warps, its outputs): without that the CTAs that got the short sequences finished last.  A share
// that begins or ends among those extra places begins or ends where the item does.
struct ArWalker {
    const AttnParams& p;
    long left;         // places of this CTA's share still to come
    int s, item, within;
    SeqInfo si;
    int tl, nt, nrb;   // of sequence s: first tile, tiles per item, row blocks

    __device__ __forceinline__ void load_seq() {
        si = seq_info(p, s);
        const KeyRange kr = key_range(p, si, 0, si.q_len);
        tl = kr.a / AR_TILE;
        nt = ar_tile_count(kr);
        nrb = (si.q_len * p.group + AR_ROWS - 1) / AR_ROWS;
    }
    __device__ __forceinline__ bool next(ArSeg& g) {
        if (left <= 0) return false;
        while (item >= nrb * p.nkv) {  // (sequences without rows have no items)
            if (++s >= p.n_seqs) return false;
            item = within = 0;
            load_seq();
        }
        if (within == 0 && left <= AR_ITEM_COST) return false;  // (its first places: the item is the next CTA's)
        if (within > 0 && within <= AR_ITEM_COST) left += within, within = 0;
        const int n = (int)min(left, (long)(nt + AR_ITEM_COST - within)), rb = item % nrb, w1 = within + n;
        g.valid = 1, g.s = s, g.q0 = si.q0, g.q_len = si.q_len, g.kv = si.kv, g.kvh = item / nrb;
        g.begins = within == 0, g.ends = w1 == nt + AR_ITEM_COST;
        g.st0 = tl + max(0, within - AR_ITEM_COST), g.st1 = tl + w1 - AR_ITEM_COST;
        left -= n, within = w1;
        g.more = nt + AR_ITEM_COST - w1;
        if (g.ends) within = 0, ++item;
        g.r0 = rb * AR_ROWS, g.n_rows = min(AR_ROWS, si.q_len * p.group - g.r0);
        const KeyRange kr = key_range(p, si, g.r0 / p.group, (g.r0 + g.n_rows - 1) / p.group + 1);
        g.t0 = max(g.st0, kr.a / AR_TILE), g.t1 = min(g.st1, (kr.b + AR_TILE - 1) / AR_TILE);
        g.a = kr.a, g.b = kr.b, g.a2 = kr.a2, g.b2 = kr.b2;
        return true;
    }
};
struct ArTiles {  // tiles of all items of a sequence
    __device__ static __forceinline__ long count(const AttnParams& p, int s) {
        const SeqInfo si = seq_info(p, s);
        const KeyRange kr = key_range(p, si, 0, si.q_len);
        return (long)((si.q_len * p.group + AR_ROWS - 1) / AR_ROWS) * p.nkv * (ar_tile_count(kr) + AR_ITEM_COST);
    }
};
// First tile of CTA c of n when `total` tiles are shared evenly
__device__ __noinline__ long ar_share(long total, int c, int n) { return total * c / n; }
// The last CTA of n whose share begins before place `end`
__device__ __noinline__ int ar_last(long total, long end, int n) { return (int)((end * n + total - 1) / total) - 1; }
constexpr int AR_MIN_TILES = 2;  // fewer tiles than this per CTA: fewer CTAs (a share of one tile costs more in joining than it saves)
__device__ __forceinline__ int ar_ctas(long total, int grid) { return (int)max(1l, min((long)grid, total / AR_MIN_TILES)); }

// The place of this CTA where up to 64 sequences are shared evenly, by one warp: each length is read once
template <typename F>
__device__ __noinline__ int plan_few(const AttnParams& p, long& total, int& n_ctas, long& share, long& before) {
    const int lane = threadIdx.x & 31;
    const long long c0 = lane < p.n_seqs ? (long long)F::count(p, lane) : 0ll, c1 = lane + 32 < p.n_seqs ? (long long)F::count(p, lane + 32) : 0ll;
    long long i0 = c0, i1 = c1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u0 = __shfl_up_sync(0xffffffffu, i0, o), u1 = __shfl_up_sync(0xffffffffu, i1, o);
        if (lane >= o) i0 += u0, i1 += u1;
    }
    i1 += __shfl_sync(0xffffffffu, i0, 31);
    total = __shfl_sync(0xffffffffu, i1, 31);
    n_ctas = ar_ctas(total, gridDim.x);
    share = ar_share(total, min((int)blockIdx.x, n_ctas), n_ctas);
    const unsigned p0 = __ballot_sync(0xffffffffu, i0 > share), p1 = __ballot_sync(0xffffffffu, i1 > share);
    if (!(p0 | p1)) return -1;
    const int f = __ffs(p0 ? p0 : p1) - 1;
    before = __shfl_sync(0xffffffffu, p0 ? i0 - c0 : i1 - c1, f);
    return p0 ? f : f + 32;
}

template <int HD, int R> struct ArScratch {  // layout of the scratch: joins, then per CTA two slots of (m, l) and outputs
    __host__ __device__ static size_t join_floats(int ctas) { return (size_t)ctas * (sizeof(ArJoin) / 4); }
    __host__ __device__ static size_t floats(int ctas) { return join_floats(ctas) + (size_t)ctas * 2 * R * (HD + 2); }
    __device__ static float* ml(float* base, int ctas, int slot) { return base + join_floats(ctas) + (size_t)slot * R * 2; }
    __device__ static float* o(float* base, int ctas, int slot) { return base + join_floats(ctas) + (size_t)ctas * 2 * R * 2 + (size_t)slot * R * HD; }
};

template <typename T, int HD>
__global__ void __launch_bounds__(AR_THREADS, ArShape<HD>::CTAS_PER_SM) attn_rows_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                                                               const __grid_constant__ AttnParams params) {
    using Sh = ArShape<HD>;
    using Scratch = ArScratch<HD, AR_ROWS>;
    constexpr int KW = AR_TILE / 4, NT = KW / 8, QPITCH = Sh::NCH * 64 + 8;
    extern __shared__ __align__(1024) uint8_t ar_raw[];
    uint8_t* sm = ar_raw + ((1024u - (smem_u32(ar_raw) & 1023u)) & 1023u);
    const uint32_t ring = smem_u32(sm);
    T* qs = reinterpret_cast<T*>(sm + (size_t)Sh::STAGES * 2 * Sh::TILE_BYTES);
    float* buf = reinterpret_cast<float*>(qs + AR_ROWS * QPITCH);  // one 16 x HD output while the warps join
    ArHeader* hdr = reinterpret_cast<ArHeader*>(reinterpret_cast<uint8_t*>(buf) + AR_ROWS * Sh::BUF_PITCH * 4);
    const AttnParams& p = hdr->p;
    volatile int* cta_abort = &hdr->abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < Sh::STAGES; ++i) mbar_init(smem_u32(&hdr->full[i]), 1), mbar_init(smem_u32(&hdr->empty[i]), 4);
        for (int i = 0; i < AR_SEGS; ++i) mbar_init(smem_u32(&hdr->seg_full[i]), 1), mbar_init(smem_u32(&hdr->seg_empty[i]), 4);
        mbar_init(smem_u32(&hdr->q_full), 1), mbar_init(smem_u32(&hdr->q_empty), 4);
        hdr->abort_flag = 0, hdr->odd = 0;
        mbar_fence_init();
    }
    if (tid < (int)(sizeof(AttnParams) / 4)) reinterpret_cast<uint32_t*>(&hdr->p)[tid] = reinterpret_cast<const uint32_t*>(&params)[tid];
    __syncthreads();
    pdl_wait_prior_grids();
    pdl_release_dependents();

    // many sequences: all threads read their lengths; few: the copying warp alone
    int n_ctas = 1, first_seq = 0;
    long total = 0, before = 0, share = 0;  // places of the whole batch, before the sequence and before this CTA's share
    if (p.n_seqs > AR_FEW_SEQS) {
        find_item<ArTiles>(p, 1l << 62, total, hdr->scan);
        n_ctas = ar_ctas(total, gridDim.x);
        share = ar_share(total, min((int)blockIdx.x, n_ctas), n_ctas);
        first_seq = find_item<ArTiles>(p, share, before, hdr->scan);
    }
    int it = 0;  // tiles so far, over all segments: stage it % STAGES

    if (warp == 4) {
        // ------------------------------------------------------------ plan and copies
        ArWalker w{p};
        if (p.n_seqs <= AR_FEW_SEQS) first_seq = plan_few<ArTiles>(p, total, n_ctas, share, before);
        w.left = 0, w.s = first_seq, w.item = w.within = w.nrb = 0;
        if (lane == 0) {
            (reinterpret_cast<ArJoin*>(p.scratch) + blockIdx.x)->n_rows = 0;
            hdr->scan[34] = total, hdr->scan[35] = n_ctas;
        }
        if (first_seq >= 0 && (int)blockIdx.x < n_ctas) {  // else: nothing for this CTA
            w.load_seq();
            w.left = ar_share(total, blockIdx.x + 1, n_ctas) - share;
            const long ahead = share - before;
            w.item = (int)(ahead / (w.nt + AR_ITEM_COST)), w.within = (int)(ahead - (long)w.item * (w.nt + AR_ITEM_COST));
        }
        int q_no = 0;
        for (int n = 0; !*cta_abort; ++n) {
            ArSeg g = {};
            const bool any = w.next(g);
            if (n >= AR_SEGS && !wait_bar(&hdr->seg_empty[n % AR_SEGS], (n / AR_SEGS - 1) & 1, DEV_TIMEOUT_EMPTY, cta_abort)) break;
            if (lane == 0) {
                hdr->seg[n % AR_SEGS] = g;
                mbar_arrive(smem_u32(&hdr->seg_full[n % AR_SEGS]));
            }
            if (!any) break;
            // queries: a row of HD elements at a time; the math warps have taken the ones before to their registers
            if (n > 0 && !wait_bar(&hdr->q_empty, (n - 1) & 1, DEV_TIMEOUT_EMPTY, cta_abort)) break;
            if (lane == 0) mbar_arrive_expect_tx(smem_u32(&hdr->q_full), (uint32_t)(g.n_rows * HD * 2));
            __syncwarp();
            q_no = n + 1;
            for (int r = lane; r < g.n_rows; r += 32) {
                const int tok = (g.r0 + r) / p.group, h = g.kvh * p.group + (g.r0 + r) - tok * p.group;
                bulk_g2s(smem_u32(qs + r * QPITCH), static_cast<const T*>(p.q) + (size_t)(g.q0 + tok) * p.q_stride + (size_t)h * HD, HD * 2, smem_u32(&hdr->q_full));
            }
            int first, count, slots = 0, pages = 0;
            if (g.t0 < g.t1) {
                tile_boxes<AR_TILE>(p, g.t0, g.a, g.b, first, count);
                pages = page_of_boxes<AR_TILE>(p, g.s, g.q0, g.t0, first, count, slots);
            }
            for (int t = g.t0; t < g.t1; ++t, ++it) {
                const int st = it % Sh::STAGES;
                int nfirst = 0, ncount = 0, npages = 0, nslots = 0;
                if (t + 1 < g.t1) {  // the next tile's pages are looked up before this tile's turn comes
                    tile_boxes<AR_TILE>(p, t + 1, g.a, g.b, nfirst, ncount);
                    npages = page_of_boxes<AR_TILE>(p, g.s, g.q0, t + 1, nfirst, ncount, nslots);
                }
                if (it >= Sh::STAGES && !wait_bar(&hdr->empty[st], ((it / Sh::STAGES) - 1) & 1, DEV_TIMEOUT_EMPTY, cta_abort)) break;
                const uint32_t bar = smem_u32(&hdr->full[st]), dst = ring + (uint32_t)st * 2 * Sh::TILE_BYTES;
                if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(count * 2 * Sh::NCH * 128) << p.box_shift);
                __syncwarp();
                load_tile<AR_TILE, Sh::NCH>(p, &kmap, dst, bar, 0, first, count, pages, slots, g.kvh);
                load_tile<AR_TILE, Sh::NCH>(p, &vmap, dst + Sh::TILE_BYTES, bar, 0, first, count, pages, slots, g.kvh);
                first = nfirst, count = ncount, pages = npages, slots = nslots;
            }
        }
        // copies in flight land before the CTA ends (after a normal run the math warps have seen them all)
        if (*cta_abort) {
#pragma unroll 1
            for (int i = max(0, it - Sh::STAGES); i <= it; ++i) {
                if (i == it && q_no == 0) break;
                const uint32_t bar = smem_u32(i < it ? &hdr->full[i % Sh::STAGES] : &hdr->q_full), ph = (i < it ? i / Sh::STAGES : q_no - 1) & 1;
                const long long c0 = clock64();
                while (!mbar_try_wait(bar, ph))
                    if (clock64() - c0 > WAIT_LIMIT_CYCLES) {
                        raise_status(DEV_TIMEOUT_DRAIN);
                        break;
                    }
            }
        }
        return;
    }

    // ---------------------------------------------------------------- math warps
    const int qr = lane >> 2, pq = lane & 3;
    const int key_w = KW * warp;  // this warp's keys of a tile
    for (int sn = 0;; ++sn) {
        // (a wait that runs out does not end a math warp's run over the segments it knows of: the warps meet at barriers; without
        // a next segment all four stop alike)
        if (!wait_bar(&hdr->seg_full[sn % AR_SEGS], (sn / AR_SEGS) & 1, DEV_TIMEOUT_FULL, cta_abort)) hdr->seg[sn % AR_SEGS].valid = 0;
        math_sync();  // (also: the buffer of the segment before has been read)
        const ArSeg& w = hdr->seg[sn % AR_SEGS];
        if (!w.valid) break;
        const int n_rows = w.n_rows, t0 = w.t0, t1 = w.t1, r0 = w.r0, pos0 = w.kv - w.q_len;
        wait_bar(&hdr->q_full, sn & 1, DEV_TIMEOUT_FULL, cta_abort);
        // this thread's two rows: the keys [lo, hi) they see
        int lo[2], hi[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = qr + 8 * e;
            const int pos = pos0 + (r0 + r) / p.group;
            hi[e] = r < n_rows ? max(pos + 1, 0) : 0;
            lo[e] = first_key(p, pos);
        }
        uint32_t qf[Sh::Q_REGS ? HD / 16 : 1][4];
        const uint32_t qa = smem_u32(qs + (lane & 15) * QPITCH + (lane >> 4) * 8);
        if constexpr (Sh::Q_REGS) {
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) ldsm_x4(qf[kk], qa + kk * 32);
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&hdr->q_empty));
        }
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        float o[HD / 8][4];
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

        for (int t = t0; t < t1; ++t, ++it) {
            const int st = it % Sh::STAGES;
            wait_bar(&hdr->full[st], (it / Sh::STAGES) & 1, DEV_TIMEOUT_FULL, cta_abort);  // (on to the end even if it runs out: the warps meet at barriers)
            const uint32_t ks = ring + (uint32_t)st * 2 * Sh::TILE_BYTES, vs = ks + Sh::TILE_BYTES;
            const int k0 = t * AR_TILE;
            const bool masked = k0 < w.a2 || k0 + AR_TILE > w.b2;  // some row does not see some key of the tile
            if (masked) {
                uint4* vp = reinterpret_cast<uint4*>(sm + (size_t)st * 2 * Sh::TILE_BYTES + Sh::TILE_BYTES);
                const int left = min(max(w.a2 - k0, 0), AR_TILE), right = min(max(w.b2 - k0, left), AR_TILE);
                bool odd = false;
#pragma unroll 1
                for (int ch = 0; ch < Sh::NCH; ++ch) {
                    if (left > 0) odd |= clear_values<T, 1>(vp + ch * AR_TILE * 8, 0, left, w.a - k0, w.b - k0, tid, 128);
                    odd |= clear_values<T, 1>(vp + ch * AR_TILE * 8, right, AR_TILE, w.a - k0, w.b - k0, tid, 128);
                }
                if (odd) hdr->odd = 1;  // (stays set: the rows of later segments are looked at too)
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the stage is refilled by a copy
                math_sync();
            }
            // scores: 16 rows x KW keys
            float sc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
                uint32_t(&a)[4] = qf[Sh::Q_REGS ? kk : 0];
                if constexpr (!Sh::Q_REGS) ldsm_x4(a, qa + kk * 32);
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    const int row = key_w + 8 * n + (lane & 7) + ((lane >> 4) & 1) * 8, c = kk * 16 + ((lane >> 3) & 1) * 8;
                    uint32_t b[4];
                    ldsm_x4(b, ks + (uint32_t)((c >> 6) * AR_TILE + row) * 128u + ((((uint32_t)(c & 63) >> 3) ^ (row & 7)) << 4));
                    mma_16<T>(sc[n], a[0], a[1], a[2], a[3], b[0], b[1]);
                    mma_16<T>(sc[n + 1], a[0], a[1], a[2], a[3], b[2], b[3]);
                }
            }
            if (masked) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = k0 + key_w + 8 * n + 2 * pq + (e & 1);
                        if (key < lo[e >> 1] || key >= hi[e >> 1]) sc[n][e] = -INFINITY;
                    }
            }
            // running softmax (m in raw scores; kq_scale > 0)
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < NT; ++n) mx[0] = fmaxf(mx[0], fmaxf(sc[n][0], sc[n][1])), mx[1] = fmaxf(mx[1], fmaxf(sc[n][2], sc[n][3]));
            bool grew = false;
            float mu[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
                mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
                grew |= mx[e] > m[e];
            }
            if (__any_sync(0xffffffffu, grew)) {
                float f[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float mn = fmaxf(m[e], mx[e]);
                    f[e] = mn == -INFINITY ? 1.f : fast_exp2((m[e] - mn) * p.scale_log2);
                    m[e] = mn, l[e] *= f[e];
                }
#pragma unroll
                for (int n = 0; n < HD / 8; ++n) o[n][0] *= f[0], o[n][1] *= f[0], o[n][2] *= f[1], o[n][3] *= f[1];
            }
            mu[0] = m[0] == -INFINITY ? 0.f : m[0], mu[1] = m[1] == -INFINITY ? 0.f : m[1];
            uint32_t pa[NT / 2][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float e0 = fast_exp2((sc[n][0] - mu[0]) * p.scale_log2), e1 = fast_exp2((sc[n][1] - mu[0]) * p.scale_log2);
                const float e2 = fast_exp2((sc[n][2] - mu[1]) * p.scale_log2), e3 = fast_exp2((sc[n][3] - mu[1]) * p.scale_log2);
                l[0] += e0 + e1, l[1] += e2 + e3;
                pa[n >> 1][(n & 1) * 2] = pack2<T>(e0, e1);
                pa[n >> 1][(n & 1) * 2 + 1] = pack2<T>(e2, e3);
            }
            // outputs: P (16 x KW) . V (KW x HD)
#pragma unroll
            for (int j = 0; j < NT / 2; ++j) {
                const int row = key_w + 16 * j + (lane & 15);
#pragma unroll
                for (int n = 0; n < HD / 8; n += 2) {
                    const int c = 8 * n + ((lane >> 4) & 1) * 8;
                    uint32_t b[4];
                    ldsm_x4_t(b, vs + (uint32_t)((c >> 6) * AR_TILE + row) * 128u + ((((uint32_t)(c & 63) >> 3) ^ (row & 7)) << 4));
                    mma_16<T>(o[n], pa[j][0], pa[j][1], pa[j][2], pa[j][3], b[0], b[1]);
                    mma_16<T>(o[n + 1], pa[j][0], pa[j][1], pa[j][2], pa[j][3], b[2], b[3]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&hdr->empty[st]));
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
        }

        if constexpr (!Sh::Q_REGS) {
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&hdr->q_empty));
        }
        // where the segment's result goes: the output rows, or a slot of scratch (0: continues an item, 1: begins one)
        const bool whole = w.begins && w.ends;
        const int slot = 2 * (int)blockIdx.x + (w.begins ? 1 : 0);
        float* sml = whole ? nullptr : Scratch::ml(p.scratch, gridDim.x, slot);
        float* so = whole ? nullptr : Scratch::o(p.scratch, gridDim.x, slot);
        auto out_elem = [&](int r) {  // element index of row r's first output
            const int tok = (r0 + r) / p.group, h = w.kvh * p.group + (r0 + r) % p.group;
            return (size_t)(w.q0 + tok) * p.out_stride + (size_t)h * HD;
        };
        auto row_sees = [&](int r) {  // row r has keys at all (else its output is 0)
            return pos0 + (r0 + r) / p.group >= 0;
        };
        {
            // the four warps' parts, added through one buffer in a fixed order
            if (pq == 0)
#pragma unroll
                for (int e = 0; e < 2; ++e) hdr->ml[warp][qr + 8 * e][0] = m[e], hdr->ml[warp][qr + 8 * e][1] = l[e];
            math_sync();
            float f[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = qr + 8 * e;
                const float mm = fmaxf(fmaxf(hdr->ml[0][r][0], hdr->ml[1][r][0]), fmaxf(hdr->ml[2][r][0], hdr->ml[3][r][0]));
                f[e] = m[e] == -INFINITY ? 0.f : fast_exp2((m[e] - mm) * p.scale_log2);
            }
#pragma unroll 1
            for (int u = 0; u < 4; ++u) {
                if (warp == u) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if (qr + 8 * e >= n_rows) continue;
                        float* row = buf + (qr + 8 * e) * Sh::BUF_PITCH + 2 * pq;
#pragma unroll
                        for (int i = 0; i < HD / 8; ++i) {
                            float2* d = reinterpret_cast<float2*>(row + 8 * i);
                            const float2 x = u == 0 ? make_float2(0.f, 0.f) : *d;
                            // (a warp without keys has zeros, which a factor of 0 keeps; one with a NaN keeps that too)
                            *d = make_float2(x.x + o[i][2 * e] * f[e], x.y + o[i][2 * e + 1] * f[e]);
                        }
                    }
                }
                math_sync();
            }
            for (int i = tid; i < n_rows * (HD / 2); i += 128) {
                const int r = i / (HD / 2), c = (i - r * (HD / 2)) * 2;
                float mm = -INFINITY, ll = 0.f;
#pragma unroll
                for (int u = 0; u < 4; ++u) mm = fmaxf(mm, hdr->ml[u][r][0]);
#pragma unroll
                for (int u = 0; u < 4; ++u) ll += hdr->ml[u][r][0] == -INFINITY ? hdr->ml[u][r][1] : hdr->ml[u][r][1] * fast_exp2((hdr->ml[u][r][0] - mm) * p.scale_log2);
                const float2 x = *reinterpret_cast<const float2*>(buf + r * Sh::BUF_PITCH + c);
                if (whole) {
                    const float inv = row_sees(r) ? 1.f / ll : 0.f;
                    store_out2(p.out, p.out_dtype, out_elem(r) + c, row_sees(r) ? x.x * inv : 0.f, row_sees(r) ? x.y * inv : 0.f);
                } else {
                    *reinterpret_cast<float2*>(so + (size_t)r * HD + c) = x;
                    if (c == 0) sml[2 * r] = mm, sml[2 * r + 1] = ll;
                }
            }
        }
        if (hdr->odd) {  // (set before the barriers above; rows by warp, once all their stores are done)
            math_sync();
            const int lo = max(w.a, w.st0 * AR_TILE), hi = min(w.b, w.st1 * AR_TILE), left = min(max(w.a2, lo), hi), right = max(min(w.b2, hi), left);
            const int ra = r0 + n_rows * warp / 4, rz = r0 + n_rows * (warp + 1) / 4;
            add_odd_values<T, HD>(p, w.s, w.q0, pos0, w.kvh, lo, left, ra, rz, so, r0);
            add_odd_values<T, HD>(p, w.s, w.q0, pos0, w.kvh, right, hi, ra, rz, so, r0);
        }
        if (w.begins && !w.ends && tid == 0) {
            // this item goes on in the next CTAs: how many of them
            ArJoin j;
            j.s = w.s, j.q0 = w.q0, j.tok_row0 = r0, j.n_rows = n_rows, j.kvh = w.kvh;
            j.any_key = pos0;  // position of token 0
            const long total = hdr->scan[34];
            const int n_ctas = (int)hdr->scan[35];
            const long item_end = ar_share(total, blockIdx.x + 1, n_ctas) + w.more;  // (a segment that does not end its item ends the share)
            j.n_parts = ar_last(total, item_end, n_ctas) - (int)blockIdx.x + 1, j.pad = 0;
            reinterpret_cast<ArJoin*>(p.scratch)[blockIdx.x] = j;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&hdr->seg_empty[sn % AR_SEGS]));
    }
}

// Adds the parts of the items that several CTAs share, in key order.  A warp per row, eight parts in flight (one after the other,
// each took a round trip to L2: 10 us for 37 parts).
template <int HD, int R>
__global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ AttnParams p, int ctas) {
    constexpr int E = HD / 32, BATCH = 8;  // elements of a lane: E lane .. E lane + E - 1
    pdl_wait_prior_grids();
    const ArJoin j = reinterpret_cast<const ArJoin*>(p.scratch)[blockIdx.x];
    const int lane = threadIdx.x & 31;
    for (int r = blockIdx.y * 4 + (threadIdx.x >> 5); r < j.n_rows; r += gridDim.y * 4) {
        auto slot_of = [&](int i) { return 2 * ((int)blockIdx.x + i) + (i == 0 ? 1 : 0); };
        auto load = [&](int i, float (&x)[E]) {
            const float* o = ArScratch<HD, R>::o(p.scratch, ctas, slot_of(i)) + (size_t)r * HD + E * lane;
            if constexpr (E % 4 == 0) {
#pragma unroll
                for (int e = 0; e < E; e += 4) {
                    const float4 v = *reinterpret_cast<const float4*>(o + e);
                    x[e] = v.x, x[e + 1] = v.y, x[e + 2] = v.z, x[e + 3] = v.w;
                }
            } else if constexpr (E == 2) {
                const float2 v = *reinterpret_cast<const float2*>(o);
                x[0] = v.x, x[1] = v.y;
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] = o[e];
            }
        };
        float x[BATCH][E];
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
            if (i < j.n_parts) load(i, x[i]);
        float mm = -INFINITY;
        for (int i = lane; i < j.n_parts; i += 32) mm = fmaxf(mm, ArScratch<HD, R>::ml(p.scratch, ctas, slot_of(i))[2 * r]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
        const float mu = mm == -INFINITY ? 0.f : mm;
        float ll = 0.f, acc[E];
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.f;
        for (int i0 = 0; i0 < j.n_parts; i0 += 32) {
            float f = 0.f, lp = 0.f;
            if (i0 + lane < j.n_parts) {
                const float* ml = ArScratch<HD, R>::ml(p.scratch, ctas, slot_of(i0 + lane)) + 2 * r;
                f = fast_exp2((ml[0] - mu) * p.scale_log2);  // (a part without keys: maximum -inf, sum 0; its factor of 0 keeps both)
                lp = ml[1] * f;
            }
            const int n = min(32, j.n_parts - i0);
            for (int b = 0; b < n; b += BATCH) {
                float y[BATCH][E];
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
#pragma unroll
                    for (int e = 0; e < E; ++e) y[i][e] = x[i][e];
                    if (i0 + b + BATCH + i < j.n_parts) load(i0 + b + BATCH + i, x[i]);  // the next batch
                }
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const float fi = __shfl_sync(0xffffffffu, f, b + i), li = __shfl_sync(0xffffffffu, lp, b + i);
                    if (b + i < n) {
                        ll += li;
#pragma unroll
                        for (int e = 0; e < E; ++e) acc[e] += y[i][e] * fi;
                    }
                }
            }
        }
        const int tok = (j.tok_row0 + r) / p.group, h = j.kvh * p.group + (j.tok_row0 + r) % p.group;
        const bool sees = j.any_key + tok >= 0;
        const float inv = 1.f / ll;
#pragma unroll
        for (int e = 0; e < E; ++e)
            store_out1(p.out, p.out_dtype, (size_t)(j.q0 + tok) * p.out_stride + (size_t)h * HD + E * lane + e, sees ? acc[e] * inv : 0.f);
    }
}

// ---- host side ----
template <typename T, int HD>
static int attn_rows_inst(const AttnParams& p, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s) {
    constexpr size_t smem = ar_smem_bytes<HD>();
    static std::mutex mu;
    static bool configured[64] = {};
    int dev = 0;
    QMM_CUDA_TRY(cudaGetDevice(&dev));
    {
        std::lock_guard<std::mutex> g(mu);
        if (dev < 0 || dev >= 64 || !configured[dev]) {
            QMM_CUDA_TRY(cudaFuncSetAttribute(attn_rows_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            if (dev >= 0 && dev < 64) configured[dev] = true;
        }
    }
    const int ctas = sm_count() * ArShape<HD>::CTAS_PER_SM;
    if (int st = launch_overlapped(attn_rows_kernel<T, HD>, dim3(ctas), dim3(AR_THREADS), smem, s, km, vm, p)) return st;
    return launch_overlapped(attn_join_kernel<HD, AR_ROWS>, dim3(ctas, AR_ROWS / 4), dim3(128), 0, s, p, ctas);
}

template <int HD> static long ar_scratch_bytes_of() { return 4 * (long)ArScratch<HD, AR_ROWS>::floats(sm_count() * ArShape<HD>::CTAS_PER_SM); }
static long attn_rows_scratch_bytes(int hd) {
    switch (hd) {
    case 32: return ar_scratch_bytes_of<32>();
    case 64: return ar_scratch_bytes_of<64>();
    case 96: return ar_scratch_bytes_of<96>();
    case 128: return ar_scratch_bytes_of<128>();
    case 256: return ar_scratch_bytes_of<256>();
    }
    return QMM_ERR_UNSUPPORTED;
}

static int attn_rows_launch(const AttnParams& p, const CUtensorMap& km, const CUtensorMap& vm, int dtype, int hd, cudaStream_t s) {
    const bool f16 = dtype == QMM_DT_F16;
    switch (hd) {
    case 32: return f16 ? attn_rows_inst<__half, 32>(p, km, vm, s) : attn_rows_inst<__nv_bfloat16, 32>(p, km, vm, s);
    case 64: return f16 ? attn_rows_inst<__half, 64>(p, km, vm, s) : attn_rows_inst<__nv_bfloat16, 64>(p, km, vm, s);
    case 96: return f16 ? attn_rows_inst<__half, 96>(p, km, vm, s) : attn_rows_inst<__nv_bfloat16, 96>(p, km, vm, s);
    case 128: return f16 ? attn_rows_inst<__half, 128>(p, km, vm, s) : attn_rows_inst<__nv_bfloat16, 128>(p, km, vm, s);
    case 256: return f16 ? attn_rows_inst<__half, 256>(p, km, vm, s) : attn_rows_inst<__nv_bfloat16, 256>(p, km, vm, s);
    }
    return QMM_ERR_UNSUPPORTED;
}

}  // namespace qmm
