// paged_attention_wide.cu - attention over the paged cache for many query rows per sequence
// (prompts, chunks of prompts), on the 5th-generation tensor cores.
//
// A tile is MT x 128 query rows (row = token * group + head of the group, so the heads that share
// keys share a tile) against blocks of 128 keys. Per block S = Q K^T and then O += P V are
// tcgen05 MMAs with M = 128; S, P and each block's P V live in TMEM.
//   * K and V come row by row through the page table: a copy that may start and end anywhere in a
//     page and that fills what is behind the last key with zeros, so it is done by a producer
//     warpgroup (16-byte cp.async for BF16; for the 8-bit formats through registers, where they
//     become binary16), in the 128-byte swizzle. K is K-major; V is the MN-major operand of P V in
//     the same layout.
//   * BF16 queries: two tiles of 128 rows share each K/V block, and one warpgroup's softmax runs
//     under the other's MMAs. P overwrites S in TMEM.
//   * F32 queries: one tile of 128 rows, its terms (hi + lo binary16; three bfloat16 terms over a
//     BF16 cache) one after another into the same accumulator, the weights the same.
//   * A softmax thread owns a row: no shuffles. It reads S twice (maximum, then weights), keeps
//     the output row in registers, and adds each block's P V to it with the FMA that rescales it,
//     so TMEM never needs a correction pass and long sequences do not add up truncated sums.
//   * 8-bit: key scales multiply S, value scales P; both come with the block in shared memory.
// Every wait is bounded; a wait that runs out raises LAI_DEVERR_TIMEOUT and ends the kernel.
#include "paged_attention.cuh"
#include "umma.cuh"

namespace lai {
namespace paged {
namespace {

using bulk::smem_addr;

constexpr int kThreads = 512;      // 2 softmax warpgroups, producers, MMA warp (+ 3 idle warps)
constexpr int kU = 128;            // keys per block
constexpr int kRing = 4;           // blocks whose scales and flags are kept
constexpr uint64_t kWaitNs = 2000000000ull;

template <int HD, int FMT, bool QF32>
struct Cfg {
    static constexpr bool kF16 = FMT != LAI_KV_BF16;
    static constexpr int kTerms = QF32 ? (kF16 ? 2 : 3) : 1;
    static constexpr int MT = QF32 ? 1 : 2;
    static constexpr int R = 128 * MT;
    static constexpr int kTile = 128 * HD * 2;  // bytes of an operand tile
    static constexpr int kStages = kF16 || QF32 ? 4 : 5;
    static constexpr float kLift = kF16 ? 13.f : 0.f;
};

template <int HD, int FMT, bool QF32>
struct Ctl {
    using C = Cfg<HD, FMT, QF32>;
    static constexpr int kScales = C::kF16 ? kU : 1;
    uint64_t full[C::kStages], empty[C::kStages];
    uint64_t info[kRing];
    uint64_t q_full[2], s_full[2], p_full[2], pv_full[2], group[2];
    float kscale[kRing][kScales], vscale[kRing][kScales];
    int vexp[kRing][4];
    int groups[kRing];  // bit i: 16-key group i of the block lies in a real page
    int vbad[kRing];    // the block (counted) from whose V infinities or NaN were taken out
    SchedSmem sched;
    uint32_t tmem;
    int abort, last[2];
};

// 128-byte swizzled tiles: [HD / 64][128 rows][128 bytes], 16-byte chunk c of row r at c ^ (r % 8).
__device__ __forceinline__ uint32_t chunk_off(int row, int chunk) {
    return (uint32_t)((chunk >> 3) * 16384 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024u >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// MN-major: 64 columns (128 bytes) of 8 k-rows are an atom; leading offset to the next 64 columns,
// stride offset to the next 8 k-rows.
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(16384u >> 4) << 16 |
           (uint64_t)(1024u >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
template <bool F16, int N, bool B_MN>
__host__ __device__ constexpr uint32_t idesc() {
    return (1u << 4) | ((F16 ? 0u : 1u) << 7) | ((F16 ? 0u : 1u) << 10) | ((B_MN ? 1u : 0u) << 16) |
           ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
        "r"(id), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b),
        "r"(id), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                 "r"(real ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t dst, const uint4 &v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z),
                 "r"(v.w)
                 : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t src) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(src)
                 : "memory");
    return v;
}
template <bool F16> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <bool F16> __device__ __forceinline__ uint32_t take2(float &x0, float &x1) {
    const uint32_t p = pack2<F16>(x0, x1);
    float f0, f1;
    if (F16)
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
            : "=f"(f0), "=f"(f1)
            : "r"(p));
    else
        f0 = bf16_lo(p), f1 = bf16_hi(p);
    x0 -= f0;
    x1 -= f1;
    return p;
}
template <bool F16> __device__ __forceinline__ bool drop_nonfinite(uint32_t &p) {
    constexpr uint32_t kLo = F16 ? 0x7c00u : 0x7f80u, kHi = kLo << 16;
    const bool lo = (p & kLo) == kLo, hi = (p & kHi) == kHi;
    p &= (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0x0000ffffu : 0xffffffffu);
    return lo || hi;
}
struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

// 8 elements of a row of q.
template <bool F32> __device__ __forceinline__ void load8(const void *p, int64_t at, float (&x)[8]) {
    if (F32) {
        float lo[4], hi[4];
        unpack<float>(__ldg(reinterpret_cast<const uint4 *>(static_cast<const float *>(p) + at)), lo);
        unpack<float>(__ldg(reinterpret_cast<const uint4 *>(static_cast<const float *>(p) + at + 4)), hi);
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = lo[e], x[4 + e] = hi[e];
    } else {
        unpack<uint16_t>(__ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + at)), x);
    }
}

// One element as F32, without its scale.
template <int FMT> __device__ __forceinline__ float element(const unsigned char *v, int64_t i) {
    if (FMT == LAI_KV_BF16) return to_f(reinterpret_cast<const uint16_t *>(v)[i]);
    if (FMT == LAI_KV_I8) return (float)reinterpret_cast<const int8_t *>(v)[i];
    const uint32_t h = e4m3x2_to_f16x2(v[i]);
    float f;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.f32.f16 %0, l;\n\t}" : "=f"(f) : "r"(h));
    return f;
}

// The items of a CTA in order; every role walks them by itself and sees the same ones.
template <int R>
struct Walk {
    using S = Sched<R, kU>;
    Range w;
    int64_t pos, slot_at, item0, item1;
    int slot, seq, head, blk0, blk1;
    Tile tl;
    __device__ __forceinline__ void start(const AttnArgs &a, const Range &r) {
        w = r;
        pos = r.w0;
        slot = r.slot;
        seq = r.seq;
        slot_at = r.at;
        if (pos < w.w1) tl = S::tile(a, slot, seq);
    }
    __device__ __forceinline__ bool next(const AttnArgs &a) {
        if (pos >= w.w1) return false;
        while (pos >= slot_at + (int64_t)tl.cost * a.kv.n_kv) {
            slot_at += (int64_t)tl.cost * a.kv.n_kv;
            if (++slot >= w.n_slots) return false;  // lengths that changed under the kernel
            while (seq + 1 < a.kv.n_seqs && S::base(a, seq + 1) <= slot) seq++;
            tl = S::tile(a, slot, seq);
        }
        head = (int)((pos - slot_at) / tl.cost);
        item0 = slot_at + (int64_t)head * tl.cost;
        item1 = item0 + tl.cost;
        blk0 = tl.b0 + (int)(pos - item0);
        const int64_t end = min(item1, w.w1);
        blk1 = tl.b0 + (int)(end - item0);
        begins = pos == item0;
        ends = item1 <= w.w1;
        pos = end;
        return true;
    }
    bool begins, ends;
    __device__ __forceinline__ int first(const AttnArgs &a) const { return tl.pos0 + tl.row0 / a.group; }
    __device__ __forceinline__ int last(const AttnArgs &a) const {
        return tl.pos0 + (tl.row0 + tl.rows - 1) / a.group;
    }
    // Rows of the tile differ in which keys of block blk they see.
    __device__ __forceinline__ bool mixed(const AttnArgs &a, int blk, int first, int last) const {
        const int jf = max(blk * kU, tl.k0), jl = min(blk * kU + kU, tl.k1) - 1;
        return jl > first || (a.window && jf <= last - a.window);
    }
};

template <int HD, int FMT, bool QF32>
__global__ void __launch_bounds__(kThreads, 1)
paged_attn_wide_kernel(void *out, const void *__restrict__ qp, const AttnArgs a) {
    using C = Cfg<HD, FMT, QF32>;
    constexpr bool kF16 = C::kF16;
    constexpr int MT = C::MT, R = C::R, kTerms = C::kTerms, ST = C::kStages;
    constexpr int kBytes = Fmt<FMT>::kBytes;
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char *q_smem = smem, *st_smem = smem + MT * kTerms * C::kTile;
    auto &ctl = *reinterpret_cast<Ctl<HD, FMT, QF32> *>(st_smem + ST * C::kTile);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wg = threadIdx.x >> 7;
    const int wt = threadIdx.x & 127;  // thread of its warpgroup
    volatile int *abort_flag = &ctl.abort;

    pdl_wait_prior();
    pdl_launch_dependents();
    if (smem_addr(smem) & 1023u) {  // the same for every thread
        if (threadIdx.x == 0) flag(a.err, LAI_DEVERR_SMEM_ALIGN);
        return;
    }
    if (blockIdx.x == 0)
        for (int s = threadIdx.x; s < a.kv.n_seqs; s += kThreads)
            if (!load_seq(a.kv, s).ok) flag(a.err, LAI_DEVERR_POSITION);
    const Range range = find_range<R, kU, kThreads>(a, ctl.sched);
    if (range.w0 >= range.w1) return;  // the whole CTA
    if (warp == 12) {
        umma::tmem_alloc(&ctl.tmem, 512);
        umma::tmem_relinquish();
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) {
            bulk::mbar_init(&ctl.full[i], 128);
            bulk::mbar_init(&ctl.empty[i], 1);
        }
        for (int i = 0; i < kRing; i++) bulk::mbar_init(&ctl.info[i], 128);
        for (int i = 0; i < kRing; i++) ctl.vbad[i] = -1;
        for (int i = 0; i < 2; i++) {
            bulk::mbar_init(&ctl.q_full[i], 128);
            bulk::mbar_init(&ctl.group[i], 128);
            bulk::mbar_init(&ctl.s_full[i], 1);
            bulk::mbar_init(&ctl.p_full[i], 128);
            bulk::mbar_init(&ctl.pv_full[i], 1);
        }
        ctl.abort = 0;
        bulk::fence_barrier_init();
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = ctl.tmem;
    // TMEM columns: S (and P over it with two tiles), P V; with one tile P has its own columns
    constexpr uint32_t kP = MT == 2 ? 0 : 128, kPV = MT == 2 ? 256 : 384;

    // Bounded wait; false once this CTA gives up. wait_warp: the whole warp, which agrees.
    auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
        if (bulk::mbar_try_wait(bar, parity)) return true;
        const uint64_t t0 = bulk::globaltimer_ns();
        for (uint32_t n = 1;; n++) {
            if (bulk::mbar_try_wait(bar, parity)) return true;
            if ((n & 63u) == 0) {
                if (*abort_flag) return false;
                if (bulk::globaltimer_ns() - t0 > kWaitNs) {
                    *abort_flag = 1;
                    flag(a.err, LAI_DEVERR_TIMEOUT);
                    return false;
                }
            }
        }
    };

    auto wait_warp = [&](uint64_t *bar, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, wait(bar, parity));
    };

    Walk<R> it;
    it.start(a, range);
    if (wg == 2) {
        // ================= producers: K and V block by block =================================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        constexpr int kIn = HD * kBytes / 16;          // 16-byte runs of a stored row
        constexpr int kRowsAtOnce = 128 / kIn;         // rows that the warpgroup loads at a time
        constexpr int kPasses = 128 / kRowsAtOnce;
        constexpr int kAhead = FMT == LAI_KV_BF16 ? ST - 2 : 0;  // cp.async tiles under way
        const int c = wt % kIn, r_in = wt / kIn;
        const int in_page = a.kv.page_size() - 1;
        uint32_t idx = 0, blocks = 0;              // operand tiles, blocks so far
        uint32_t mixed_bits = 0;                   // bit i: the tile i before the newest is a mixed V
        bool ok = true;
        // a cp.async tile has landed: mend it if it must be, and hand it over
        auto publish = [&](uint32_t i, bool mixed_v) {
            if (mixed_v) {
                bool bad = false;
                const uint32_t base = smem_addr(st_smem + (i % ST) * C::kTile);
#pragma unroll 1
                for (int p = 0; p < kPasses; p++) {
                    const uint32_t at = base + chunk_off(p * kRowsAtOnce + r_in, c);
                    uint4 v = ld_shared16(at);
                    bool b = drop_nonfinite<false>(v.x);
                    b |= drop_nonfinite<false>(v.y);
                    b |= drop_nonfinite<false>(v.z);
                    b |= drop_nonfinite<false>(v.w);
                    if (b) st_shared16(at, v);
                    bad |= b;
                }
                if (bad) ctl.vbad[(i / 2) % kRing] = (int)(i / 2);
            }
            bulk::fence_proxy_async_smem();
            bulk::mbar_arrive(&ctl.full[i % ST]);
        };
        while (ok && it.next(a)) {
            const int first = it.first(a), last = it.last(a);
            // ---- K and V
            for (int blk = it.blk0; ok && blk < it.blk1; blk++) {
                const int j0 = blk * kU;
                // lane i < 8 of every warp looks up the page of 16-key group i
                int page = -1;
                if (lane < 8 && j0 + 16 * lane < it.tl.k1) {
                    page = __ldg(a.kv.pages + (int64_t)it.tl.seq * a.kv.max_pages +
                                 ((j0 + 16 * lane) >> a.kv.log_page));
                    if (page < 0 || page >= a.kv.n_pages) {
                        if (wt < 8 && j0 + 16 * lane + 16 > it.tl.k0) flag(a.err, LAI_DEVERR_PAGE);
                        page = -1;
                    }
                }
                const int groups = (int)(__ballot_sync(0xffffffffu, page >= 0) & 0xffu);
                const bool mixed = FMT != LAI_KV_I8 && it.mixed(a, blk, first, last);
                const int slot = blocks % kRing;
                const int j_mine = j0 + wt;  // this thread's key for the scales
#pragma unroll 1
                for (int kv = 0; kv < 2; kv++, idx++) {
                    if (idx >= (uint32_t)ST && !wait_warp(&ctl.empty[idx % ST], (idx / ST - 1) & 1)) {
                        ok = false;
                        break;
                    }
                    if (kv == 0) {  // the block's scales and pages: its ring entry is free by now
                        if (kF16) {
                            const int pg = __shfl_sync(0xffffffffu, page, (wt >> 4) & 7);
                            float ks = 0.f, vs = 0.f;
                            if (pg >= 0 && j_mine >= it.tl.k0 && j_mine < it.tl.k1) {
                                const int64_t at = a.kv.page_base(pg, it.head) + (j_mine & in_page);
                                ks = __ldg(a.kv.k_scale + at);
                                vs = __ldg(a.kv.v_scale + at);
                            }
                            ctl.kscale[slot][kF16 ? wt : 0] = ks;
                            ctl.vscale[slot][kF16 ? wt : 0] = vs;
                            const uint32_t u = __float_as_uint(vs) & 0x7fffffffu;
                            const uint32_t top = __reduce_max_sync(0xffffffffu, u < 0x7f800000u ? u : 0u);
                            if (lane == 0) ctl.vexp[slot][wt >> 5] = (int)(top >> 23) - 127;
                        }
                        if (wt == 0) ctl.groups[slot] = groups;
                        bulk::mbar_arrive(&ctl.info[slot]);
                    }
                    const unsigned char *src = (kv ? a.kv.v : a.kv.k) + c * 16;
                    const uint32_t dst = smem_addr(st_smem + (idx % ST) * C::kTile);
                    if constexpr (FMT == LAI_KV_BF16) {
#pragma unroll
                        for (int p = 0; p < kPasses; p++) {
                            const int r = p * kRowsAtOnce + r_in, j = j0 + r;
                            const int pg = __shfl_sync(0xffffffffu, page, p * kRowsAtOnce / 16);
                            const bool real = pg >= 0 && j >= it.tl.k0 && j < it.tl.k1;
                            const int64_t at = a.kv.page_base(real ? pg : 0, it.head) + (real ? j & in_page : 0);
                            cp_async16(dst + chunk_off(r, c), src + at * (HD * 2), real);
                        }
                        cp_async_commit();
                        mixed_bits = mixed_bits << 1 | (uint32_t)(mixed && kv);
                        if (idx >= (uint32_t)kAhead) {
                            cp_async_wait<kAhead>();
                            publish(idx - kAhead, mixed_bits >> kAhead & 1);
                        }
                    } else {
                        uint4 raw[kPasses];
#pragma unroll
                        for (int p = 0; p < kPasses; p++) {
                            const int r = p * kRowsAtOnce + r_in, j = j0 + r;
                            // rows p * kRowsAtOnce + r_in of one warp may span two groups (HD 64)
                            const int pg = __shfl_sync(0xffffffffu, page, r >> 4);
                            raw[p] = make_uint4(0, 0, 0, 0);
                            if (pg >= 0 && j >= it.tl.k0 && j < it.tl.k1)
                                raw[p] = ld_stream(src + (a.kv.page_base(pg, it.head) + (j & in_page)) * HD);
                        }
                        bool bad = false;
#pragma unroll
                        for (int p = 0; p < kPasses; p++) {
                            const int r = p * kRowsAtOnce + r_in;
                            uint4 lo = make_uint4(half2_of<FMT, false>(raw[p].x), half2_of<FMT, true>(raw[p].x),
                                                  half2_of<FMT, false>(raw[p].y), half2_of<FMT, true>(raw[p].y));
                            uint4 hi = make_uint4(half2_of<FMT, false>(raw[p].z), half2_of<FMT, true>(raw[p].z),
                                                  half2_of<FMT, false>(raw[p].w), half2_of<FMT, true>(raw[p].w));
                            if (mixed && kv) {
                                bad |= drop_nonfinite<true>(lo.x) | drop_nonfinite<true>(lo.y) |
                                       drop_nonfinite<true>(lo.z) | drop_nonfinite<true>(lo.w);
                                bad |= drop_nonfinite<true>(hi.x) | drop_nonfinite<true>(hi.y) |
                                       drop_nonfinite<true>(hi.z) | drop_nonfinite<true>(hi.w);
                            }
                            st_shared16(dst + chunk_off(r, 2 * c), lo);
                            st_shared16(dst + chunk_off(r, 2 * c + 1), hi);
                        }
                        if (bad) ctl.vbad[slot] = (int)blocks;
                        bulk::fence_proxy_async_smem();
                        bulk::mbar_arrive(&ctl.full[idx % ST]);
                    }
                }
                blocks++;
            }
        }
        if constexpr (FMT == LAI_KV_BF16) {
            cp_async_wait<0>();
            if (ok)
                for (uint32_t i = idx < (uint32_t)kAhead ? 0 : idx - kAhead; i < idx; i++)
                    publish(i, mixed_bits >> (idx - 1 - i) & 1);
        }
    } else if (wg == 3) {
        // ================= the MMA thread ====================================================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == 12 && lane == 0) {
            constexpr uint32_t kIdS = idesc<kF16, 128, false>(), kIdO = idesc<kF16, HD, true>();
            uint32_t idx = 0, n_q[2] = {0, 0}, n_mt[2] = {0, 0};
            bool ok = true;
            auto scores = [&](int mt, uint32_t i) {
                const uint32_t kb = smem_addr(st_smem + (i % ST) * C::kTile);
#pragma unroll
                for (int t = 0; t < kTerms; t++) {
                    const uint32_t qb = smem_addr(q_smem) + (t * MT + mt) * C::kTile;
#pragma unroll
                    for (int k = 0; k < HD / 16; k++) {
                        const uint32_t off = (k / 4) * 16384 + (k % 4) * 32;
                        mma_ss(tmem + mt * 128, desc_kmajor(qb + off), desc_kmajor(kb + off), kIdS, t || k);
                    }
                }
                umma::commit(&ctl.s_full[mt]);
            };
            while (ok && it.next(a)) {
                const int tiles = MT == 2 && it.tl.rows > 128 ? 2 : 1;
                const int nb = it.blk1 - it.blk0;
                ok = wait(&ctl.full[idx % ST], (idx / ST) & 1);
                for (int mt = 0; ok && mt < tiles; mt++) {
                    ok = wait(&ctl.q_full[mt], n_q[mt]++ & 1);
                    umma::fence_after_sync();
                    if (ok) scores(mt, idx);
                }
                if (!ok) break;
                umma::commit(&ctl.empty[idx % ST]);
                for (int b = 0; ok && b < nb; b++) {
                    const uint32_t vi = idx + 1, ki = idx + 2;
                    const bool more = b + 1 < nb;
                    for (int mt = 0; ok && mt < tiles; mt++) {
                        ok = wait(&ctl.p_full[mt], n_mt[mt] & 1);
                        n_mt[mt]++;
                        if (MT == 1 && ok && more) {  // the next scores while P V waits for V
                            ok = wait(&ctl.full[ki % ST], (ki / ST) & 1);
                            umma::fence_after_sync();
                            if (ok) scores(mt, ki);
                        }
                        ok = ok && wait(&ctl.full[vi % ST], (vi / ST) & 1);
                        if (!ok) break;
                        umma::fence_after_sync();
                        const uint32_t vb = smem_addr(st_smem + (vi % ST) * C::kTile);
#pragma unroll
                        for (int t = 0; t < kTerms; t++)
#pragma unroll
                            for (int k = 0; k < kU / 16; k++)
                                mma_ts(tmem + kPV + mt * 128, tmem + kP + mt * 128 + t * 64 + k * 8,
                                       desc_mnmajor(vb + k * 2048), kIdO, t || k);
                        umma::commit(&ctl.pv_full[mt]);
                        if (MT == 2 && more) {
                            ok = wait(&ctl.full[ki % ST], (ki / ST) & 1);
                            umma::fence_after_sync();
                            if (ok) scores(mt, ki);
                        }
                    }
                    if (!ok) break;
                    umma::commit(&ctl.empty[vi % ST]);
                    if (more) umma::commit(&ctl.empty[ki % ST]);
                    idx += 2;
                }
            }
            // Every MMA is done before TMEM is given back: each result was waited for. After an
            // abort nobody waits, so the MMAs in flight get a millisecond.
            if (!ok) {
                const uint64_t t0 = bulk::globaltimer_ns();
                while (bulk::globaltimer_ns() - t0 < 1000000ull) {}
            }
        }
    } else if (wg < MT) {
        // ================= softmax: a thread per row =========================================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
        const int mt = wg;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + lane_base + mt * 128, t_p = t_s + kP, t_pv = tmem + lane_base + kPV + mt * 128;
        uint32_t n = 0, blocks = 0, n_group = 0;  // this tile's blocks, all blocks, joins
        bool ok = true;
        auto join = [&]() {  // all of the warpgroup, within the bound
            bulk::mbar_arrive(&ctl.group[mt]);
            return wait_warp(&ctl.group[mt], n_group++ & 1);
        };
        while (ok && it.next(a)) {
            const int nb = it.blk1 - it.blk0;
            if (it.tl.rows <= mt * 128) {  // no rows of this tile
                blocks += nb;
                continue;
            }
            const int r = mt * 128 + wt, fr = it.tl.row0 + r, tok = fr / a.group;
            const bool row_ok = r < it.tl.rows;
            const int row_pos = row_ok ? it.tl.pos0 + tok : -1;
            const int row_from = a.window ? row_pos - a.window : -1;  // sees (row_from, row_pos]
            const int first = it.first(a), last = it.last(a);
            float c = a.scale_log2;
            {  // this row of Q into shared memory; the last scores of the item before are done
                const int64_t at = ((int64_t)it.tl.q_row0 + tok) * a.ld_q +
                                   (int64_t)(it.head * a.group + (fr - tok * a.group)) * HD;
                const uint32_t dst = smem_addr(q_smem) + mt * C::kTile;
                float up = 1.f;
                if (kF16) {  // the row's largest into [2^13, 2^14)
                    uint32_t top = 0;
                    if (row_ok)
#pragma unroll 4
                        for (int d = 0; d < HD; d += 8) {
                            float x[8];
                            load8<QF32>(qp, at + d, x);
#pragma unroll
                            for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
                        }
                    const int e = (int)(top >> 23) - 127;
                    up = pow2i(13 - e);
                    c *= pow2i(e - 13);
                }
#pragma unroll 4
                for (int d = 0; d < HD; d += 8) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = 0.f;
                    if (row_ok) load8<QF32>(qp, at + d, x);
                    if (kF16)
#pragma unroll
                        for (int e = 0; e < 8; e++) x[e] *= up;
#pragma unroll
                    for (int t = 0; t < kTerms; t++) {
                        uint4 v;
                        v.x = take2<kF16>(x[0], x[1]);
                        v.y = take2<kF16>(x[2], x[3]);
                        v.z = take2<kF16>(x[4], x[5]);
                        v.w = take2<kF16>(x[6], x[7]);
                        st_shared16(dst + t * MT * C::kTile + chunk_off(wt, d / 8), v);
                    }
                }
                bulk::fence_proxy_async_smem();
                bulk::mbar_arrive(&ctl.q_full[mt]);
            }
            float m = neg_inf(), l = 0.f, alpha = 0.f, o[HD];
            int ve = -90;
            bool bad = false;
#pragma unroll
            for (int d = 0; d < HD; d++) o[d] = 0.f;
            auto add_pv = [&](uint32_t block) {
                umma::fence_after_sync();
#pragma unroll
                for (int g = 0; g < HD / 32; g++) {
                    uint32_t x[32];
                    umma::tmem_ld_32x32b_x32(t_pv + 32 * g, x);
                    umma::tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        o[32 * g + i] = fmaf(o[32 * g + i], alpha, __uint_as_float(x[i]));
                }
                umma::fence_before_sync();
                if (FMT != LAI_KV_I8) bad |= *(volatile int *)&ctl.vbad[block % kRing] == (int)block;
            };
            for (int b = 0; b < nb; b++, n++, blocks++) {
                const int blk = it.blk0 + b, slot = blocks % kRing;
                ok = wait_warp(&ctl.info[slot], (blocks / kRing) & 1) && wait_warp(&ctl.s_full[mt], n & 1);
                if (!ok) break;
                umma::fence_after_sync();
                const int groups = ctl.groups[slot];
                // element i of the block is seen where lo <= i <= hi
                const int hi = row_pos - blk * kU, lo = row_from + 1 - blk * kU;
                const bool masked = groups != 0xff || blk * kU + kU - 1 > first || it.tl.k0 > blk * kU ||
                                    (a.window && blk * kU <= last - a.window) || it.tl.rows < mt * 128 + 128;
                auto seen = [&](int i) { return i <= hi && i >= lo && (groups >> (i >> 4) & 1); };
                // ---- the maximum
                float top = neg_inf();
                auto max_pass = [&](auto mask) {
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        uint32_t x[32];
                        umma::tmem_ld_32x32b_x32(t_s + 32 * g, x);
                        umma::tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            float v = __uint_as_float(x[i]);
                            if (kF16) v *= ctl.kscale[slot][kF16 ? 32 * g + i : 0];
                            if (decltype(mask)::value) v = seen(32 * g + i) ? v : neg_inf();
                            top = fmaxf(top, v);
                        }
                    }
                };
                if (masked) max_pass(Yes{}); else max_pass(No{});
                if (MT == 1 && b > 0) {  // P V of the block before, while S waited
                    ok = wait_warp(&ctl.pv_full[mt], (n - 1) & 1);
                    if (!ok) break;
                    add_pv(blocks - 1);
                }
                const float mn = fmaxf(m, top == neg_inf() ? top : top * c);
                const float mu = mn == neg_inf() ? 0.f : mn;
                alpha = ex2(m - mu);
                m = mn;
                float off = mu - C::kLift;
                if (kF16) {  // sums and weights are in units of 2^ve, the largest value scale so far
                    const int *e4 = ctl.vexp[slot];
                    const int e = min(max(max(max(e4[0], e4[1]), max(e4[2], e4[3])), ve), 90);
                    alpha *= pow2i(ve - e);
                    ve = e;
                    off += (float)e;
                }
                l *= alpha;
                // ---- the weights
                float sum0 = 0.f, sum1 = 0.f;
                auto p_pass = [&](auto mask) {
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        uint32_t x[32];
                        umma::tmem_ld_32x32b_x32(t_s + 32 * g, x);
                        umma::tmem_wait_ld();
                        uint32_t w[kTerms][16];
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            float p[2];
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                float v = __uint_as_float(x[i + h]);
                                if (kF16) v *= ctl.kscale[slot][kF16 ? 32 * g + i + h : 0];
                                v = ex2(fmaf(v, c, -off));
                                if (decltype(mask)::value) v = seen(32 * g + i + h) ? v : 0.f;
                                (h ? sum1 : sum0) += v;
                                if (kF16) {
                                    const float vs = ctl.vscale[slot][kF16 ? 32 * g + i + h : 0];
                                    v = decltype(mask)::value ? (seen(32 * g + i + h) ? v * vs : 0.f) : v * vs;
                                }
                                p[h] = v;
                            }
#pragma unroll
                            for (int t = 0; t < kTerms; t++) w[t][i / 2] = take2<kF16>(p[0], p[1]);
                        }
#pragma unroll
                        for (int t = 0; t < kTerms; t++) tmem_st_x16(t_p + t * 64 + 16 * g, w[t]);
                    }
                };
                if (masked) p_pass(Yes{}); else p_pass(No{});
                l += sum0 + sum1;
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                umma::fence_before_sync();
                bulk::mbar_arrive(&ctl.p_full[mt]);
                if (MT == 2) {
                    ok = wait_warp(&ctl.pv_full[mt], n & 1);
                    if (!ok) break;
                    add_pv(blocks);
                }
            }
            if (!ok) break;
            if (MT == 1) {
                ok = wait_warp(&ctl.pv_full[mt], (n - 1) & 1);
                if (!ok) break;
                add_pv(blocks - 1);
            }
            // infinities and NaN that were taken out of blocks whose rows differ in what they see
            if (FMT != LAI_KV_I8 && bad) {
                for (int j = max(it.blk0 * kU, it.tl.k0); j < min(it.blk1 * kU, it.tl.k1); j++) {
                    if (!it.mixed(a, j / kU, first, last) || j > row_pos || j <= row_from) continue;
                    const int page = __ldg(a.kv.pages + (int64_t)it.tl.seq * a.kv.max_pages + (j >> a.kv.log_page));
                    if (page < 0 || page >= a.kv.n_pages) continue;
                    const int64_t at = (a.kv.page_base(page, it.head) + (j & (a.kv.page_size() - 1))) * HD;
#pragma unroll
                    for (int d = 0; d < HD; d++) {
                        const float v = element<FMT>(a.kv.v, at + d);
                        if ((__float_as_uint(v) & 0x7f800000u) == 0x7f800000u) o[d] += v;
                    }
                }
            }
            if (kF16) {  // back to plain units for the join: weights relative to exp2(m) alone
                const float unit = pow2i(ve);
                l *= unit;
#pragma unroll
                for (int d = 0; d < HD; d++) o[d] *= unit;
            }
            bool write = it.begins && it.ends;
            if (!write) {
                // parts: [row] max, [row] sum, then [d / 4][row][4]
                constexpr int64_t kPart = (int64_t)R * (HD + 2);
                float *pp = a.parts + ((int64_t)blockIdx.x * 2 + (it.begins ? 1 : 0)) * kPart;
                pp[r] = m;
                pp[R + r] = l;
#pragma unroll
                for (int d = 0; d < HD; d += 4)
                    *reinterpret_cast<float4 *>(pp + 2 * R + ((d / 4) * R + r) * 4) =
                        make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]);
                __threadfence();
                if (!(ok = join())) break;
                const int c0 = cta_of(it.w, it.item0), c1 = cta_of(it.w, it.item1 - 1);
                if (wt == 0) ctl.last[mt] = atomicAdd(a.counters + c0 * MT + mt, 1) == c1 - c0;
                if (!(ok = join())) break;
                write = *(volatile int *)&ctl.last[mt];
                if (write) {
                    __threadfence();
                    if (wt == 0) a.counters[c0 * MT + mt] = 0;  // ready for the next call
                    m = neg_inf();
                    l = 0.f;
#pragma unroll
                    for (int d = 0; d < HD; d++) o[d] = 0.f;
                    for (int cc = c0; cc <= c1; cc++) {
                        const float *pc = a.parts + ((int64_t)cc * 2 + (cc == c0 ? 1 : 0)) * kPart;
                        const float cm = __ldcg(pc + r), mx = fmaxf(m, cm);
                        const float mu = mx == neg_inf() ? 0.f : mx;
                        const float ca = ex2(m - mu), cb = ex2(cm - mu);
                        l = fmaf(__ldcg(pc + R + r), cb, l * ca);
                        m = mx;
#pragma unroll
                        for (int d = 0; d < HD; d += 4) {
                            const float4 v = __ldcg(reinterpret_cast<const float4 *>(pc + 2 * R + ((d / 4) * R + r) * 4));
                            o[d] = fmaf(v.x, cb, o[d] * ca);
                            o[d + 1] = fmaf(v.y, cb, o[d + 1] * ca);
                            o[d + 2] = fmaf(v.z, cb, o[d + 2] * ca);
                            o[d + 3] = fmaf(v.w, cb, o[d + 3] * ca);
                        }
                    }
                }
            }
            if (write && row_ok) {
                const int64_t at = (((int64_t)it.tl.q_row0 + tok) * ((int64_t)a.kv.n_kv * a.group) +
                                    it.head * a.group + (fr - tok * a.group)) * HD;
                const float inv = l == 0.f ? 0.f : 1.f / l;
                if (QF32) {
                    float *dst = static_cast<float *>(out) + at;
#pragma unroll
                    for (int d = 0; d < HD; d += 4)
                        *reinterpret_cast<float4 *>(dst + d) =
                            make_float4(o[d] * inv, o[d + 1] * inv, o[d + 2] * inv, o[d + 3] * inv);
                } else {
                    uint16_t *dst = static_cast<uint16_t *>(out) + at;
#pragma unroll
                    for (int d = 0; d < HD; d += 8) {
                        const float y[8] = {o[d] * inv, o[d + 1] * inv, o[d + 2] * inv, o[d + 3] * inv,
                                            o[d + 4] * inv, o[d + 5] * inv, o[d + 6] * inv, o[d + 7] * inv};
                        st_vec(dst + d, pack<uint16_t>(y));
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    if (warp == 12) umma::tmem_dealloc(tmem, 512);
}

template <int HD, int FMT, bool QF32>
int launch_wide(void *out, const void *q, const AttnArgs &a, cudaStream_t st) {
    using C = Cfg<HD, FMT, QF32>;
    constexpr size_t kSmem = (size_t)(C::MT * C::kTerms + C::kStages) * C::kTile + sizeof(Ctl<HD, FMT, QF32>);
    static_assert(kSmem <= 227 * 1024, "one CTA's shared memory");
    auto kern = paged_attn_wide_kernel<HD, FMT, QF32>;
    // the warpgroups' register shares (setmaxnreg) add up to what the block is launched with
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, kern) != cudaSuccess || fa.numRegs != 128) return LAI_ERR_CUDA;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem) != cudaSuccess)
        return LAI_ERR_CUDA;
    launch_pdl(kern, dim3(kSMs), dim3(kThreads), kSmem, st, out, q, a);
    return launch_status();
}

}  // namespace

size_t wide_scratch_floats(int head_dim) { return (size_t)kSMs * 2 * 256 * (head_dim + 2); }

int attention_wide(void *out, const void *q, bool f32, int head_dim, int format, const AttnArgs &a,
                   cudaStream_t st) {
#define LAI_WIDE(HD, FMT) (f32 ? launch_wide<HD, FMT, true>(out, q, a, st) : launch_wide<HD, FMT, false>(out, q, a, st))
    if (head_dim == 128) {
        switch (format) {
            case LAI_KV_BF16: return LAI_WIDE(128, LAI_KV_BF16);
            case LAI_KV_E4M3: return LAI_WIDE(128, LAI_KV_E4M3);
            default: return LAI_WIDE(128, LAI_KV_I8);
        }
    }
    switch (format) {
        case LAI_KV_BF16: return LAI_WIDE(64, LAI_KV_BF16);
        case LAI_KV_E4M3: return LAI_WIDE(64, LAI_KV_E4M3);
        default: return LAI_WIDE(64, LAI_KV_I8);
    }
#undef LAI_WIDE
}

}  // namespace paged
}  // namespace lai
