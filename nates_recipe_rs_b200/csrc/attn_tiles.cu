// Attention of many rows over a paged cache or over packed prompts on tcgen05: pieces of prompts and whole prompts, head_dim 64,
// 96 and 128.  Same operator and same conventions as attn_rows.cu.
//
// A CTA owns up to two tiles of 128 rows of one kv head; a row is a (token, query head of the group) pair, tokens outermost, so
// one tile of keys and values serves every query head that shares it and a tile spans few positions (128 / group tokens: little
// of the causal triangle is computed and thrown away).  For every tile of 128 keys and each of the two row tiles
//     S = Q K^T    128 x 128 x HD, both operands in shared memory, S in tensor memory (f32)
//     P = exp2((S - m) * c), row sums            one thread per row, S read with tcgen05.ld, P written back over S (16 bit)
//     O += P V     128 x HD x 128, P from tensor memory, V from shared memory as it arrives (keys are the K dimension: the
//                  operand is "MN major"), O in tensor memory for the whole run over the keys
// While the threads of one row tile compute exponentials the tensor cores work for the other: the two pipes (16 exponentials per
// clock and SM; 8192 flops) need about the same time at HD = 128.  The running maximum that P is scaled by is only moved when a
// row's maximum has grown by more than 2^8 (P <= 256 fits f16, l and O are f32): O is rescaled in tensor memory a few times per
// run instead of once per tile, with no separate correction step.
// Warps: 0-3 and 4-7 softmax of row tile 0 / 1 (and its epilogue); 8 issues the tcgen05.mma; 9 issues the TMA copies (queries,
// and keys and values through a ring of 128-key slots); 10-11 clear what no row sees out of the value tiles that need it.
// Every wait is bounded; on expiry the CTA records a status code, drains its copies, frees its tensor memory and returns.
#include "attn_pages.cuh"

namespace qmm {

constexpr int AT_TILE = 128;  // keys per tile, and rows per tile
constexpr int AT_THREADS = 384;
constexpr int AT_MAX_ROWS = 256;  // rows of an item
template <int HD> struct AtShape {
    static constexpr int NCH = (HD + 63) / 64;
    static constexpr int TILE_BYTES = NCH * AT_TILE * 128;  // 128 rows of one matrix
    static constexpr int SLOTS = NCH == 1 ? 10 : 5;         // 160 KB of keys and values
    __host__ __device__ static constexpr uint32_t IDESC_S(bool bf16) { return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | ((AT_TILE >> 3) << 17) | ((128 >> 4) << 24); }
    __host__ __device__ static constexpr uint32_t IDESC_O(bool bf16) { return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (1u << 16) | ((HD >> 3) << 17) | ((128 >> 4) << 24); }
};
constexpr uint32_t AT_COL_S = 0, AT_COL_O = 256;  // tensor memory columns: S (and P over it) of tile i at 128 i, O at 256 + 128 i

struct __align__(16) AtHeader {
    uint64_t full[10], empty[10];
    uint64_t v_ask, v_ok, q_full, q_empty, s_full[2], p_full[2], o_full[2], drain;
    long long scan[36];
    uint32_t tmem_base;
    int abort_flag, nonfinite;
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
// 128 columns of this warp's 32 lanes.  The wait is part of the statement: between a load and its wait nothing may touch the
// registers, not even a spill that the compiler puts there.
__device__ __forceinline__ void tmem_ld128(uint32_t taddr, uint32_t (&r)[128]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x128.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
        "%28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, "
        "%54, %55, %56, %57, %58, %59, %60, %61, %62, %63, %64, %65, %66, %67, %68, %69, %70, %71, %72, %73, %74, %75, %76, %77, %78, %79, "
        "%80, %81, %82, %83, %84, %85, %86, %87, %88, %89, %90, %91, %92, %93, %94, %95, %96, %97, %98, %99, %100, %101, %102, %103, %104, "
        "%105, %106, %107, %108, %109, %110, %111, %112, %113, %114, %115, %116, %117, %118, %119, %120, %121, %122, %123, %124, %125, %126"
        ", %127"
        "}, [%128];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : QMM_R8(r, 0), QMM_R8(r, 8), QMM_R8(r, 16), QMM_R8(r, 24), QMM_R8(r, 32), QMM_R8(r, 40), QMM_R8(r, 48), QMM_R8(r, 56), QMM_R8(r, 64), QMM_R8(r, 72), QMM_R8(r, 80), QMM_R8(r, 88), QMM_R8(r, 96), QMM_R8(r, 104), QMM_R8(r, 112), QMM_R8(r, 120)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::QMM_RI8(r, 0),
                 QMM_RI8(r, 8), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
        "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::QMM_RI8(r, 0),
        QMM_RI8(r, 8), QMM_RI8(r, 16), QMM_RI8(r, 24), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}

// The segments (item, tiles [t0, t1) of it) of this CTA.  An item is (sequence, kv head, block of tb tokens); where the tiles are
// shared evenly, every item of a sequence counts as many as the sequence's last block has, at least one.
struct AtWalker {
    const AttnParams& p;
    int tb;        // tokens per block
    long g, g1;
    int s, item, within;
    SeqInfo si;
    int tl, nt, nb;
    // the current segment
    int kvh, tok0, tok1, t0, t1;  // tokens [tok0, tok1), tiles [t0, t1) that hold keys of its rows
    int st0, st1;                 // tiles of the segment before that cut
    bool begins, ends;
    KeyRange kr;

    __device__ static __forceinline__ int count(const SeqInfo& si, const KeyRange& kr) {
        return max(1, (max(kr.b, 0) + AT_TILE - 1) / AT_TILE - kr.a / AT_TILE);
    }
    __device__ __forceinline__ void load_seq() {
        si = seq_info(p, s);
        const KeyRange r = key_range(p, si, 0, si.q_len);
        tl = r.a / AT_TILE;
        nt = count(si, r);
        nb = (si.q_len + tb - 1) / tb;
    }
    __device__ static __forceinline__ long tiles_of(const AttnParams& p, int tb, int s) {
        const SeqInfo si = seq_info(p, s);
        return (long)((si.q_len + tb - 1) / tb) * p.nkv * count(si, key_range(p, si, 0, si.q_len));
    }
    __device__ __forceinline__ bool next() {
        if (g >= g1) return false;
        while (item >= nb * p.nkv) {
            if (++s >= p.n_seqs) return false;
            item = within = 0;
            load_seq();
        }
        const int n = (int)min(g1 - g, (long)(nt - within));
        kvh = item / nb;
        tok0 = (item - kvh * nb) * tb, tok1 = min(tok0 + tb, si.q_len);
        st0 = tl + within, st1 = st0 + n;
        begins = within == 0, ends = within + n == nt;
        kr = key_range(p, si, tok0, tok1);
        t0 = max(st0, kr.a / AT_TILE), t1 = min(st1, (kr.b + AT_TILE - 1) / AT_TILE);
        g += n, within += n;
        if (within == nt) within = 0, ++item;
        return true;
    }
    // some row of the segment does not see some key of tile t
    __device__ __forceinline__ bool masked(int t) const { return t * AT_TILE < kr.a2 || (t + 1) * AT_TILE > kr.b2; }
};

template <typename T, int HD>
__global__ void __launch_bounds__(AT_THREADS, 1) attn_tiles_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                                                                   const __grid_constant__ CUtensorMap vmap, const __grid_constant__ AttnParams p) {
    using Sh = AtShape<HD>;
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ __align__(1024) uint8_t at_raw[];
    uint8_t* sm = at_raw + ((1024u - (smem_u32(at_raw) & 1023u)) & 1023u);
    const uint32_t q_s = smem_u32(sm), ring = q_s + 2 * Sh::TILE_BYTES;
    AtHeader* hdr = reinterpret_cast<AtHeader*>(sm + (size_t)(2 + Sh::SLOTS) * Sh::TILE_BYTES);
    volatile int* cta_abort = &hdr->abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int tpt = AT_TILE / p.group, tile_rows = tpt * p.group;  // tokens and rows of a row tile

    if (tid == 0) {
        for (int i = 0; i < Sh::SLOTS; ++i) mbar_init(smem_u32(&hdr->full[i]), 1), mbar_init(smem_u32(&hdr->empty[i]), 1);
        mbar_init(smem_u32(&hdr->v_ask), 1), mbar_init(smem_u32(&hdr->v_ok), 2);
        mbar_init(smem_u32(&hdr->q_full), 1), mbar_init(smem_u32(&hdr->q_empty), 1), mbar_init(smem_u32(&hdr->drain), 1);
        for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&hdr->s_full[i]), 1), mbar_init(smem_u32(&hdr->p_full[i]), 4), mbar_init(smem_u32(&hdr->o_full[i]), 1);
        hdr->abort_flag = 0, hdr->nonfinite = 0;
        mbar_fence_init();
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&hdr->tmem_base)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_wait_prior_grids();
    pdl_release_dependents();

    AtWalker w{p, 2 * tpt};
    int n_ctas = 1;
    long total = 0, before = 0;
    bool any;
    if (p.stream_k) {
        find_item(p.n_seqs, 1l << 62, [&](int s) { return AtWalker::tiles_of(p, 2 * tpt, s); }, total, hdr->scan);
        n_ctas = ar_ctas(total, gridDim.x);
        if (tid == 0) (reinterpret_cast<ArJoin*>(p.scratch) + blockIdx.x)->n_rows = 0;
        w.g = ar_share(total, min((int)blockIdx.x, n_ctas), n_ctas), w.g1 = ar_share(total, min((int)blockIdx.x + 1, n_ctas), n_ctas);
        w.s = find_item(p.n_seqs, w.g, [&](int s) { return AtWalker::tiles_of(p, 2 * tpt, s); }, before, hdr->scan);
        any = (int)blockIdx.x < n_ctas && w.s >= 0;
        if (any) {
            w.load_seq();
            w.item = (int)((w.g - before) / w.nt), w.within = (int)((w.g - before) % w.nt);
        }
    } else {
        // one item per CTA: block blockIdx.y of all blocks (a sequence's last, longest, first), kv head blockIdx.x
        w.s = find_item(p.n_seqs, blockIdx.y, [&](int s) { return (long)((seq_info(p, s).q_len + 2 * tpt - 1) / (2 * tpt)); }, before, hdr->scan);
        any = w.s >= 0;
        if (any) {
            w.load_seq();
            w.g = 0, w.g1 = w.nt, w.within = 0;
            w.item = blockIdx.x * w.nb + (w.nb - 1 - (int)(blockIdx.y - before));
        }
    }
    if (!any) w.g = w.g1 = 0;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = hdr->tmem_base;

    auto give_up = [&](int code) {
        if (!*cta_abort) {
            raise_status(code);
            *cta_abort = 1;
        }
    };
    auto wait = [&](uint64_t* bar, uint32_t phase, int code) {
        if (mbar_wait_bounded(smem_u32(bar), phase & 1u, cta_abort)) return true;
        give_up(code);
        return false;
    };


    if (warp == 9) {
        // ------------------------------------------------------------ copies
        int it = 0, q_no = 0;  // tiles (of keys and of values) and query blocks so far
        bool ok = true;
        while (ok && w.next()) {
            if (w.t0 >= w.t1) continue;
            const int nq = w.tok1 - w.tok0 > tpt ? 2 : 1;
            if (q_no > 0 && !wait(&hdr->q_empty, q_no - 1, DEV_TIMEOUT_EMPTY)) break;
            if (lane == 0) mbar_arrive_expect_tx(smem_u32(&hdr->q_full), (uint32_t)(nq * Sh::NCH * tile_rows * 128));
            __syncwarp();
            if (lane < nq * Sh::NCH) {
                const int i = lane / Sh::NCH, c = lane % Sh::NCH;
                tma_load_3d(q_s + (uint32_t)(i * Sh::TILE_BYTES + c * AT_TILE * 128), &qmap, c * 64, w.kvh * p.group, w.si.q0 + w.tok0 + i * tpt,
                            smem_u32(&hdr->q_full));
            }
            ++q_no;
            int first, cnt, pages;
            tile_boxes<AT_TILE>(p, w.t0, w.kr.a, w.kr.b, first, cnt);
            pages = page_of_boxes<AT_TILE>(p, w.s, w.t0, first, cnt);
            for (int t = w.t0; t < w.t1 && ok; ++t) {
                int nfirst = 0, ncnt = 0, npages = 0;
                if (t + 1 < w.t1) {  // the next tile's pages are looked up before its turn comes
                    tile_boxes<AT_TILE>(p, t + 1, w.kr.a, w.kr.b, nfirst, ncnt);
                    npages = page_of_boxes<AT_TILE>(p, w.s, t + 1, nfirst, ncnt);
                }
#pragma unroll
                for (int kv = 0; kv < 2; ++kv, ++it) {
                    const int sl = it % Sh::SLOTS;
                    if (it >= Sh::SLOTS && !wait(&hdr->empty[sl], it / Sh::SLOTS - 1, DEV_TIMEOUT_EMPTY)) {
                        ok = false;
                        break;
                    }
                    const uint32_t bar = smem_u32(&hdr->full[sl]);
                    if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)cnt * Sh::NCH * p.box_rows * 128);
                    __syncwarp();
                    load_tile<AT_TILE, Sh::NCH>(p, kv ? &vmap : &kmap, ring + (uint32_t)sl * Sh::TILE_BYTES, bar, t, first, cnt, pages, w.si.q0, w.kvh);
                }
                first = nfirst, cnt = ncnt, pages = npages;
            }
        }
        if (*cta_abort) {  // copies in flight land before the CTA ends
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
    } else if (warp == 8) {
        // ------------------------------------------------------------ tensor cores (one thread)
        if (lane == 0) {
            int it = 0, q_no = 0;
            uint32_t n_p[2] = {0, 0};  // P tiles awaited so far, per row tile
            uint32_t n_v = 0;          // value tiles handed to the clearing warps so far
            bool ok = true;
            auto mma_s = [&](int i, int slot) {
                const uint64_t qd = umma_desc_sw128(q_s + (uint32_t)i * Sh::TILE_BYTES), kd = umma_desc_sw128(ring + (uint32_t)slot * Sh::TILE_BYTES);
#pragma unroll
                for (int k16 = 0; k16 < HD / 16; ++k16) {  // 32 bytes of a 128-byte row each; the next 64 elements one chunk further
                    const uint64_t off = (uint64_t)((k16 >> 2) * (AT_TILE * 128 >> 4) + (k16 & 3) * 2);
                    umma_bf16(tmem + AT_COL_S + 128u * i, qd + off, kd + off, Sh::IDESC_S(BF16), k16 > 0);
                }
                umma_commit(smem_u32(&hdr->s_full[i]));
            };
            auto mma_o = [&](int i, int slot, bool acc) {
                const uint64_t vd = umma_desc_v(ring + (uint32_t)slot * Sh::TILE_BYTES);
#pragma unroll
                for (int k16 = 0; k16 < AT_TILE / 16; ++k16)  // 16 keys: 8 columns of P, 2048 bytes of V
                    umma_ts(tmem + AT_COL_O + 128u * i, tmem + AT_COL_S + 128u * i + 8u * k16, vd + (uint64_t)(k16 * (2048 >> 4)), Sh::IDESC_O(BF16),
                            (acc || k16 > 0) ? 1u : 0u);
            };
            // a value tile with keys that some row does not see goes through the clearing warps while its scores are in softmax
            auto ask_v = [&](int t, int v_it) {
                if (!w.masked(t)) return true;
                if (!wait(&hdr->full[v_it % Sh::SLOTS], v_it / Sh::SLOTS, DEV_TIMEOUT_FULL)) return false;
                mbar_arrive(smem_u32(&hdr->v_ask));
                ++n_v;
                return true;
            };
            while (ok && w.next()) {
                if (w.t0 >= w.t1) continue;
                const int nq = w.tok1 - w.tok0 > tpt ? 2 : 1;
                if (!wait(&hdr->q_full, q_no, DEV_TIMEOUT_FULL)) break;
                ++q_no;
                int sl = it % Sh::SLOTS;
                if (!wait(&hdr->full[sl], it / Sh::SLOTS, DEV_TIMEOUT_FULL)) break;
                tc_fence_after();
                for (int i = 0; i < nq; ++i) mma_s(i, sl);
                umma_commit(smem_u32(&hdr->empty[sl]));
                if (w.t0 + 1 == w.t1) umma_commit(smem_u32(&hdr->q_empty));
                ++it;
                ok = ask_v(w.t0, it);
                for (int t = w.t0; t < w.t1 && ok; ++t) {
                    const int vs = it % Sh::SLOTS, ks = (it + 1) % Sh::SLOTS;
                    const bool more = t + 1 < w.t1;
                    ok = wait(&hdr->full[vs], it / Sh::SLOTS, DEV_TIMEOUT_FULL);
                    if (ok && w.masked(t)) ok = wait(&hdr->v_ok, n_v - 1, DEV_TIMEOUT_FULL);
                    if (ok && more) ok = wait(&hdr->full[ks], (it + 1) / Sh::SLOTS, DEV_TIMEOUT_FULL);
                    for (int i = 0; i < nq && ok; ++i) {
                        ok = wait(&hdr->p_full[i], n_p[i], DEV_TIMEOUT_MMA);
                        if (!ok) break;
                        ++n_p[i];
                        tc_fence_after();
                        mma_o(i, vs, t > w.t0);
                        if (more) mma_s(i, ks);
                        else umma_commit(smem_u32(&hdr->o_full[i]));
                    }
                    if (!ok) break;
                    umma_commit(smem_u32(&hdr->empty[vs]));
                    if (more) {
                        umma_commit(smem_u32(&hdr->empty[ks]));
                        if (t + 2 == w.t1) umma_commit(smem_u32(&hdr->q_empty));
                    }
                    it += more ? 2 : 1;
                    if (more) ok = ask_v(t + 1, it);
                }
            }
            if (*cta_abort) {  // what was issued retires before the tensor memory is freed
                umma_commit(smem_u32(&hdr->drain));
                const long long c0 = clock64();
                while (!mbar_try_wait(smem_u32(&hdr->drain), 0))
                    if (clock64() - c0 > WAIT_LIMIT_CYCLES) {
                        raise_status(DEV_TIMEOUT_DRAIN);
                        break;
                    }
            }
        }
        __syncwarp();
    } else if (warp >= 10) {
        // ------------------------------------------------------------ value tiles with keys that some row does not see
        // Values that no row sees become zeros; where some row does not see a key, a value that is not finite does too (the
        // tensor cores would add 0 * it), and the segment's rows are computed again by attn_row_exact.
        // The issuing thread asks for each such tile when it has landed and waits for it before it asks for the next: these
        // warps do not follow the ring's own barriers, most of whose phases they would skip.
        int it = 0;
        uint32_t n_v = 0;
        bool ok = true;
        while (ok && w.next()) {
            for (int t = w.t0; t < w.t1; ++t, it += 2) {
                if (!w.masked(t)) continue;
                const int sl = (it + 1) % Sh::SLOTS;
                if (!wait(&hdr->v_ask, n_v++, DEV_TIMEOUT_FULL)) {
                    ok = false;
                    break;
                }
                uint4* vp = reinterpret_cast<uint4*>(sm + (size_t)(2 + sl) * Sh::TILE_BYTES);
                const int k0 = t * AT_TILE;
                bool odd = false;
                for (int i = tid - 320; i < Sh::NCH * AT_TILE * 8; i += 64) {
                    const int key = k0 + ((i >> 3) % AT_TILE);
                    if (key >= w.kr.a2 && key < w.kr.b2) continue;
                    bool clear = key < w.kr.a || key >= w.kr.b;
                    if (!clear) {
                        const uint4 y = vp[i];
                        clear = has_nonfinite<T>(y.x) || has_nonfinite<T>(y.y) || has_nonfinite<T>(y.z) || has_nonfinite<T>(y.w);
                        odd |= clear;
                    }
                    if (clear) vp[i] = make_uint4(0u, 0u, 0u, 0u);
                }
                if (odd) *reinterpret_cast<volatile int*>(&hdr->nonfinite) = 1;  // (stays set: later segments of the CTA go the exact way too)
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // read by the tensor cores, refilled by a copy
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&hdr->v_ok));
            }
        }
    } else {
        // ------------------------------------------------------------ softmax and epilogue: a thread per row
        const int wg = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + AT_COL_S + 128u * wg, to = tmem + lanes + AT_COL_O + 128u * wg;
        uint32_t n_s = 0, n_o = 0;
        const float c = p.scale_log2;
        const bool vec = reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && (p.out_stride * (p.out_dtype == QMM_DT_F32 ? 4 : 2)) % 16 == 0;
        bool ok = true;
        while (ok && w.next()) {
            const int n_tok = w.tok1 - w.tok0, tok = w.tok0 + wg * tpt + row / p.group;
            if (wg * tpt >= n_tok) continue;  // no rows in this row tile
            const bool live = row < tile_rows && tok < w.tok1;
            const int pos = w.si.kv - w.si.q_len + tok;
            const int hi = live ? max(pos + 1, 0) : 0, lo = p.window ? max(0, pos - p.window + 1) : 0;
            float m = -INFINITY, l = 0.f;
            for (int t = w.t0; t < w.t1; ++t) {
                if (!wait(&hdr->s_full[wg], n_s, DEV_TIMEOUT_MMA)) {
                    ok = false;
                    break;
                }
                ++n_s;
                tc_fence_after();
                uint32_t sr[4][32];  // the row
#pragma unroll
                for (int q = 0; q < 4; ++q) tmem_ld32(ts + 32 * q, sr[q]);
                if (w.masked(t)) {
                    const int k0 = t * AT_TILE;
#pragma unroll
                    for (int j = 0; j < AT_TILE; ++j)
                        if (k0 + j < lo || k0 + j >= hi) sr[j >> 5][j & 31] = 0xFF800000u;  // -inf
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < AT_TILE; j += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(sr[j >> 5][(j & 31) + 2 * e]), __uint_as_float(sr[j >> 5][(j & 31) + 2 * e + 1]));
                const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                if (t == w.t0) {
                    m = mt;
                } else {
                    const bool grew = (mt - m) * c > 8.f || (m == -INFINITY && mt > -INFINITY);
                    if (__any_sync(0xffffffffu, grew)) {
                        const float mn = fmaxf(m, mt), f = mn == -INFINITY ? 1.f : fast_exp2((m - mn) * c);
                        m = mn, l *= f;
#pragma unroll 1
                        for (int q = 0; q < HD / 32; ++q) {
                            uint32_t r[32];
                            tmem_ld32(to + 32 * q, r);
#pragma unroll
                            for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * f);
                            tmem_st32(to + 32 * q, r);
                        }
                    }
                }
                const float mc = m == -INFINITY ? 0.f : m * c;
                float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t pk[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float e0 = fast_exp2(fmaf(__uint_as_float(sr[q][2 * j]), c, -mc)), e1 = fast_exp2(fmaf(__uint_as_float(sr[q][2 * j + 1]), c, -mc));
                        ls[j & 1] += e0, ls[2 + (j & 1)] += e1;
                        pk[j] = pack2<T>(e0, e1);
                    }
                    tmem_st16(ts + 16 * q, pk);
                }
                l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&hdr->p_full[wg]));
            }
            if (!ok) break;
            if (w.t0 < w.t1) {
                if (!wait(&hdr->o_full[wg], n_o, DEV_TIMEOUT_MMA)) break;
                ++n_o;
                tc_fence_after();
            }
            const bool whole = w.begins && w.ends;
            const int slot = 2 * (int)blockIdx.x + (w.begins ? 1 : 0), r = (tok - w.tok0) * p.group + row % p.group;  // row of the item
            const int head = w.kvh * p.group + row % p.group;
            float* ml = whole ? nullptr : ArScratch<HD, AT_MAX_ROWS>::ml(p.scratch, gridDim.x, slot);
            float* so = whole ? nullptr : ArScratch<HD, AT_MAX_ROWS>::o(p.scratch, gridDim.x, slot);
            const size_t oe = (size_t)(w.si.q0 + tok) * p.out_stride + (size_t)head * HD;
            if (*reinterpret_cast<volatile int*>(&hdr->nonfinite)) {
                // a row at a time by the whole warp
                for (int u = 0; u < 32; ++u) {
                    const int rr = (warp & 3) * 32 + u, tk = w.tok0 + wg * tpt + rr / p.group, ps = w.si.kv - w.si.q_len + tk, hd = w.kvh * p.group + rr % p.group;
                    if (rr >= tile_rows || tk >= w.tok1) break;
                    float em, el, eo[HD / 32];
                    attn_row_exact<T, HD>(p, w.s, w.si.q0, tk, hd, w.kvh, max(w.st0 * AT_TILE, p.window ? max(0, ps - p.window + 1) : 0),
                                          min(w.st1 * AT_TILE, ps + 1), em, el, eo);
                    const int r2 = (tk - w.tok0) * p.group + rr % p.group;
                    const float inv = 1.f / el;
#pragma unroll
                    for (int j = 0; j < HD / 32; ++j) {
                        if (whole) store_out1(p.out, p.out_dtype, (size_t)(w.si.q0 + tk) * p.out_stride + (size_t)hd * HD + lane + 32 * j, ps >= 0 ? eo[j] * inv : 0.f);
                        else so[(size_t)r2 * HD + lane + 32 * j] = eo[j];
                    }
                    if (!whole && lane == 0) ml[2 * r2] = em, ml[2 * r2 + 1] = el;
                }
            } else {
                const bool sees = pos >= 0;
                const float inv = 1.f / l;
#pragma unroll 1
                for (int q = 0; q < HD / 32; ++q) {
                    uint32_t o[32];
                    if (w.t0 < w.t1) {
                        tmem_ld32(to + 32 * q, o);
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = 0u;
                    }
                    if (live) {
                        if (!whole) {
#pragma unroll
                            for (int j = 0; j < 32; j += 4)
                                *reinterpret_cast<uint4*>(so + (size_t)r * HD + 32 * q + j) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] = sees ? __float_as_uint(__uint_as_float(o[j]) * inv) : 0u;
                            if (vec && p.out_dtype == QMM_DT_F32) {
#pragma unroll
                                for (int j = 0; j < 32; j += 4)
                                    *reinterpret_cast<uint4*>(static_cast<float*>(p.out) + oe + 32 * q + j) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                            } else if (vec) {
                                uint32_t h[16];
#pragma unroll
                                for (int j = 0; j < 16; ++j) {
                                    const float a = __uint_as_float(o[2 * j]), b = __uint_as_float(o[2 * j + 1]);
                                    h[j] = p.out_dtype == QMM_DT_F16 ? pack2<__half>(a, b) : pack2<__nv_bfloat16>(a, b);
                                }
#pragma unroll
                                for (int j = 0; j < 16; j += 4)
                                    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + oe + 32 * q + 2 * j) = make_uint4(h[j], h[j + 1], h[j + 2], h[j + 3]);
                            } else {
#pragma unroll
                                for (int j = 0; j < 32; j += 2) store_out2(p.out, p.out_dtype, oe + 32 * q + j, __uint_as_float(o[j]), __uint_as_float(o[j + 1]));
                            }
                        }
                    }
                }
                if (!whole && live) ml[2 * r] = m, ml[2 * r + 1] = l;
            }
            if (w.begins && !w.ends && tid == 0) {  // this item goes on in the next CTAs: how many of them
                ArJoin j;
                j.s = w.s, j.q0 = w.si.q0, j.tok_row0 = w.tok0 * p.group, j.n_rows = n_tok * p.group, j.kvh = w.kvh;
                j.any_key = w.si.kv - w.si.q_len;
                const long item_end = w.g1 + (w.nt - (w.st1 - w.tl));
                int e = blockIdx.x + 1;
                while (ar_share(total, e + 1, n_ctas) < item_end) ++e;
                j.n_parts = e - (int)blockIdx.x + 1, j.pad = 0;
                reinterpret_cast<ArJoin*>(p.scratch)[blockIdx.x] = j;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
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
    const int tb = 2 * (AT_TILE / p.group), ctas = sm_count();
    const long blocks = (long)p.total_q / tb + p.n_seqs;  // at least as many as there are
    if (!p.stream_k && blocks > 65535) return QMM_ERR_UNSUPPORTED;
    if (int st = launch_overlapped(attn_tiles_kernel<T, HD>, p.stream_k ? dim3(ctas) : dim3(p.nkv, (unsigned)blocks), dim3(AT_THREADS), smem, s, qm, km, vm, p)) return st;
    if (p.stream_k) return launch_overlapped(attn_join_kernel<HD, AT_MAX_ROWS>, dim3(ctas, AT_MAX_ROWS / 4), dim3(128), 0, s, p, ctas);
    return QMM_OK;
}
static bool attn_tiles_fits(int hd) { return hd == 64 || hd == 96 || hd == 128; }
static long attn_tiles_scratch_bytes(int hd) {
    return 4 * (long)(hd == 64 ? ArScratch<64, AT_MAX_ROWS>::floats(sm_count()) : hd == 96 ? ArScratch<96, AT_MAX_ROWS>::floats(sm_count()) : ArScratch<128, AT_MAX_ROWS>::floats(sm_count()));
}
// The queries as (element, head, row), a box = the rows of one row tile: tokens outermost, the heads of a group inside
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
    if (hd == 64) return f16 ? attn_tiles_inst<__half, 64>(p, qm, km, vm, s) : attn_tiles_inst<__nv_bfloat16, 64>(p, qm, km, vm, s);
    if (hd == 96) return f16 ? attn_tiles_inst<__half, 96>(p, qm, km, vm, s) : attn_tiles_inst<__nv_bfloat16, 96>(p, qm, km, vm, s);
    return f16 ? attn_tiles_inst<__half, 128>(p, qm, km, vm, s) : attn_tiles_inst<__nv_bfloat16, 128>(p, qm, km, vm, s);
}

}  // namespace qmm
