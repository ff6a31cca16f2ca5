// paged_attention_wide.cu - attention over the paged cache for many query rows per sequence
// (prompts, chunks of prompts), on the 5th-generation tensor cores.
//
// A tile is MT x 128 query rows (row = token * group + head of the group, so the heads that share
// keys share a tile) against blocks of 128 keys. Per block S = Q K^T and then O += P V are
// tcgen05 MMAs with M = 128; S, P and O (or a block's P V) live in TMEM.
//   * One warp brings K and V through the page table, 16 keys at a time (a page holds a multiple
//     of 16): BF16 with TMA tensor copies straight into the MMA's 128-byte swizzle, the 8-bit
//     formats (and their scales) with bulk copies into a staging ring. A second warpgroup finishes
//     each tile: it turns 8-bit values into binary16, and writes zeros over values behind the last
//     key. K is K-major; V is the MN-major operand of P V in the same layout.
//   * BF16 queries: two tiles of 128 rows share each K/V block, and one warpgroup's softmax runs
//     under the other's MMAs. A softmax thread owns a row (no shuffles) and holds the block's 128
//     scores in registers; P overwrites S in TMEM. The maximum that weights are relative to only
//     moves when it has grown by 2^8, so O is hardly ever rescaled.
//   * F32 queries: one tile of 128 rows, whose softmax the two warpgroups share (a thread of each
//     per row, for half of the block's keys and half of the output's columns), its terms (hi + lo
//     binary16; three bfloat16 terms over a BF16 cache) one after another into the same
//     accumulator, smallest first, the weights the same. A block's P V starts from zero and is
//     added to the output row, which the threads keep in registers, so long sequences do not add
//     up the MMA's truncated sums.
//   * 8-bit: key scales multiply S, value scales P; both come with the block in shared memory.
//     Weights are relative to the row's largest product of a weight and a value's scale, so that they
//     fit binary16 and neither a value that the row does not see nor a large one under a small weight
//     costs it bits. Where a block's scales lie within 2^kSpread the largest stands for all of them;
//     elsewhere every key's own counts.
// Measured, 2048 tokens over 32768 keys, 16 heads of 128 on 8 (0.53 TFLOP of products below the
// diagonal): BF16 q, BF16 cache 474 us (1.12 PFLOP/s, 0.67 of a large BF16 matrix product's rate),
// 8-bit 580 to 590 us; F32 q 1575 us (BF16 cache) and 1230 us (8-bit), for three and two times the
// products of each kind; runs differ by 5% with the power cap. With BF16 q softmax and MMAs bound it
// together: a tile's block is 16384 exponentials, 1024 clocks at 16 per SM and clock, and its MMAs take
// as many; 8-bit caches have room for 3 operand tiles only, so conversions are not far enough ahead of
// the MMAs (BF16 with 3 tiles: 525 us).
// Every wait is bounded; a wait that runs out raises LAI_DEVERR_TIMEOUT and ends the kernel.
#include <cuda.h>

#include <mutex>

#include "paged_attention.cuh"
#include "umma.cuh"

namespace lai {
namespace paged {
namespace {

using bulk::smem_addr;

constexpr int kThreads = 512;  // 2 softmax warpgroups, finishers, MMA warp, copy warp (+ 2 idle)
constexpr int kU = 128;        // keys per block
constexpr int kGroup = 16;     // keys per copy
constexpr int kRing = 4;       // blocks whose scales and flags are kept
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr float kGrow = 8.f;   // log2 of how far weights may pass 1 before O is rescaled
constexpr int kSpread = 12;    // log2 of how far a block's value scales lie apart at most, to go by the largest
// log2 of the value scales that sums of weights have room for: weights reach from 2^kLift over the
// scale, with 2^-24 of it still a normal F32, to 2^20 times 2^14 over it
constexpr int kLowScale = -90, kTopScale = 106;

template <int HD, int FMT, bool QF32>
struct Cfg {
    static constexpr bool kF16 = FMT != LAI_KV_BF16;
    static constexpr int kTerms = QF32 ? (kF16 ? 2 : 3) : 1;
    static constexpr int MT = QF32 ? 1 : 2;
    static constexpr int R = 128 * MT;
    static constexpr int kTile = 128 * HD * 2;         // bytes of an operand tile
    // What fits beside the queries. BF16 q over 2048 x 32768 keys: BF16 keys 525, 463, 464 us with 3, 4
    // and 5 tiles; INT8 keys 582 and 608 us with 3 tiles and 3 or 2 in the staging ring, 857 with 4 and 1.
    static constexpr int kStages = kF16 || QF32 ? 3 : 5;
    static constexpr int kRaw = kF16 ? 3 : 0;          // 8-bit tiles in the staging ring
    static constexpr int kRawTile = 128 * HD;
    static constexpr int kLand = kF16 ? kRaw : kStages;  // tiles that copies land in
    // binary16 weights: 2^kLift at the row's maximum, at most 2^14 with kGrow (two tiles) and a value
    // scale's mantissa, so that small ones are held to 2^-25 of 2^kLift (of 2^(kLift - kSpread), where
    // the block's largest scale is not that of the row's largest product)
    static constexpr float kLift = !kF16 ? 0.f : QF32 ? 13.f : 5.f;
    using S = Sched<R, kU, 3>;
};

// A CTA's part of an item, as the copy warp hands it to the other roles.
struct Item {
    int seq, head, row0, rows, q_row0, pos0;  // rows 0: no more items
    int first, last, k0, k1;                  // positions of its first and last row; keys any row sees
    int blk0, blk1;                           // this CTA's blocks
    int c0, c1;                               // the CTAs that have a part of it
    bool begins, whole;                       // has its first block; has all of them
};
constexpr int kItems = 4;  // items under way

template <int HD, int FMT, bool QF32>
struct Ctl {
    using C = Cfg<HD, FMT, QF32>;
    static constexpr int kScales = C::kF16 ? kU : 4;
    float kscale[kRing][kScales], vscale[kRing][kScales];  // 16-byte aligned
    float swap[QF32 ? 2 : 1][2][QF32 ? 128 : 1];           // between the halves of a row
    uint64_t landed[C::kLand], taken[C::kLand], full[C::kStages], empty[C::kStages];
    uint64_t info[kRing], item_full[kItems], item_empty[kItems];
    Item items[kItems];
    uint64_t q_full[2], s_full[2], p_full[2][2], pv_full[2], group[2];
    uint32_t vspan[kRing][4];  // of 32 keys' value scales the largest exponent, and 255 less the smallest
    int groups[kRing];  // bit i: 16-key group i of the block lies in a real page
    int vbad[kRing];    // the block (counted) from whose V infinities or NaN were taken out
    SeqSmem seqs;
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
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap *map, int x, int y,
                                            uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_addr(bar))
        : "memory");
}
// The largest of three, NaN if one of them is.
__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}
struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };


// One element as F32, without its scale.
template <int FMT> __device__ __forceinline__ float element(const unsigned char *v, int64_t i) {
    if (FMT == LAI_KV_BF16) return to_f(reinterpret_cast<const uint16_t *>(v)[i]);
    if (FMT == LAI_KV_I8) return (float)reinterpret_cast<const int8_t *>(v)[i];
    const uint32_t h = e4m3x2_to_f16x2(v[i]);
    float f;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.f32.f16 %0, l;\n\t}" : "=f"(f) : "r"(h));
    return f;
}

template <int HD, int FMT, bool QF32>
__global__ void __launch_bounds__(kThreads, 1)
paged_attn_wide_kernel(void *out, const void *__restrict__ qp, const AttnArgs a,
                       const __grid_constant__ CUtensorMap k_map,
                       const __grid_constant__ CUtensorMap v_map) {
    using C = Cfg<HD, FMT, QF32>;
    using S = typename C::S;
    constexpr bool kF16 = C::kF16;
    constexpr int MT = C::MT, R = C::R, kTerms = C::kTerms, ST = C::kStages, LD = C::kLand;
    constexpr int kBytes = Fmt<FMT>::kBytes;
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char *q_smem = smem, *st_smem = smem + MT * kTerms * C::kTile;
    unsigned char *raw_smem = st_smem + ST * C::kTile;
    auto &ctl = *reinterpret_cast<Ctl<HD, FMT, QF32> *>(raw_smem + C::kRaw * C::kRawTile);
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int wg = warp >> 2, wt = threadIdx.x & 127;  // warpgroup, thread of it

    pdl_wait_prior();
    pdl_launch_dependents();
    if (smem_addr(smem) & 1023u) {  // the same for every thread
        if (threadIdx.x == 0) flag(a.err, LAI_DEVERR_SMEM_ALIGN);
        return;
    }
    const AttnArgs as = cache_seqs<kThreads>(a, ctl.seqs);
    if (as.kv.n_seqs == 0) return;  // the whole grid
    // (in the place of Q, which comes behind the barrier below)
    const Range range = find_range<S, kThreads>(as, *reinterpret_cast<SchedSmem *>(q_smem));
    if (range.w0 >= range.w1) return;  // the whole CTA
    if (warp == 12) {
        umma::tmem_alloc(&ctl.tmem, 512);
        umma::tmem_relinquish();
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < LD; i++) {
            bulk::mbar_init(&ctl.landed[i], 1);
            bulk::mbar_init(&ctl.taken[i], 4);
        }
        for (int i = 0; i < ST; i++) {
            bulk::mbar_init(&ctl.full[i], 4);
            bulk::mbar_init(&ctl.empty[i], 1);
        }
        for (int i = 0; i < kRing; i++) {
            bulk::mbar_init(&ctl.info[i], 4);
            ctl.vbad[i] = -1;
        }
        for (int i = 0; i < kItems; i++) {
            bulk::mbar_init(&ctl.item_full[i], 1);
            bulk::mbar_init(&ctl.item_empty[i], 4 + 1 + 8);
        }
        for (int i = 0; i < 2; i++) {
            bulk::mbar_init(&ctl.q_full[i], 256 / MT);
            bulk::mbar_init(&ctl.group[i], 256 / MT);
            bulk::mbar_init(&ctl.s_full[i], 1);
            bulk::mbar_init(&ctl.p_full[i][0], 128);
            bulk::mbar_init(&ctl.p_full[i][1], 128);
            bulk::mbar_init(&ctl.pv_full[i], 1);
        }
        ctl.abort = 0;
        bulk::fence_barrier_init();
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = ctl.tmem;
    // TMEM columns: S (and P over it with two tiles), then O or a block's P V; with one tile P has
    // its own columns
    constexpr uint32_t kP = MT == 2 ? 0 : 128, kPV = MT == 2 ? 256 : 384;

    // Bounded wait of a whole warp, which agrees on the answer; false when it ran out.
    auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
        bool ok = bulk::mbar_try_wait(bar, parity);
        if (!ok) {
            const uint64_t t0 = bulk::globaltimer_ns();
            do
                ok = bulk::mbar_try_wait(bar, parity);
            while (!ok && bulk::globaltimer_ns() - t0 < kWaitNs);
            if (!ok) ctl.abort = 1;
        }
        return __all_sync(0xffffffffu, ok);
    };

    // The next item for a warp of any role but the copies'; false at the end.
    uint32_t n_items = 0;
    Item it;
    auto next = [&](bool &ok) -> bool {
        const uint32_t i = n_items % kItems;
        if (!(ok = wait(&ctl.item_full[i], (n_items / kItems) & 1))) return false;
        n_items++;
        it = ctl.items[i];
        __syncwarp();
        if (lane == 0) bulk::mbar_arrive(&ctl.item_empty[i]);
        return it.rows != 0;
    };
    // The page of 16-key group `lane` (< 8) of the block at j0, or -1.
    auto page_of = [&](int seq, int k1, int j0) -> int {
        const int j = j0 + kGroup * lane;
        if (lane >= kU / kGroup || j >= k1) return -1;
        const int page = __ldg(a.kv.pages + (int64_t)seq * a.kv.max_pages + (j >> a.kv.log_page));
        return page >= 0 && page < a.kv.n_pages ? page : -1;
    };
    const int in_page = a.kv.page_size() - 1;

    // Register shares: 2 x 128 x 192 + 2 x 128 x 64 = 512 x 128
    if (wg < 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");

    if (warp == 13) {
        // ================= copies ============================================================
        uint32_t idx = 0, blocks = 0;  // operand tiles, blocks so far
        bool ok = true;
        Walk<S> w;
        w.start(as, range);
        for (;;) {
            const bool more = w.next(as);
            const Tile &tl = w.tl;
            const int head = w.kv_head();
            const uint32_t slot = n_items % kItems;
            if (n_items >= kItems && !(ok = wait(&ctl.item_empty[slot], (n_items / kItems - 1) & 1))) break;
            n_items++;
            if (lane == 0) {
                Item &to = ctl.items[slot];
                to = Item{tl.seq, head, tl.row0, more ? tl.rows : 0, tl.q_row0, tl.pos0, tl.first, tl.last,
                          tl.k0, tl.k1, w.blk0, w.blk1, 0, 0, w.begins, w.begins && w.ends};
                if (more && !to.whole) {
                    to.c0 = range.cta_of(w.item0);
                    to.c1 = range.cta_of(w.item1 - 1);
                }
                bulk::mbar_arrive(&ctl.item_full[slot]);
            }
            __syncwarp();
            if (!more) break;
            for (int r = lane; r < tl.rows; r += 32) {  // the item's queries on their way to L2
                const int fr = tl.row0 + r, tok = a.by_group.of(fr);
                const char *q = static_cast<const char *>(qp) +
                                (((int64_t)tl.q_row0 + tok) * a.ld_q +
                                 (int64_t)(head * a.group + (fr - tok * a.group)) * HD) * (QF32 ? 4 : 2);
#pragma unroll
                for (int i = 0; i < HD * (QF32 ? 4 : 2); i += 128)
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(q + i));
            }
            for (int blk = w.blk0; ok && blk < w.blk1; blk++, blocks++) {
                const int j0 = blk * kU;
                const int page = page_of(tl.seq, tl.k1, j0);
                const uint32_t groups = __ballot_sync(0xffffffffu, page >= 0);
                for (int kv = 0; kv < 2; kv++, idx++) {
                    const uint32_t land = idx % LD;
                    if (idx >= (uint32_t)LD &&
                        !(ok = wait(kF16 ? &ctl.taken[land] : &ctl.empty[land], (idx / LD - 1) & 1)))
                        break;
                    constexpr uint32_t kGroupBytes = kGroup * HD * kBytes;
                    if (lane == 0) {
                        const uint32_t n = __popc(groups);
                        bulk::mbar_arrive_expect_tx(&ctl.landed[land],
                                                    n * (kGroupBytes + (kF16 && kv == 0 ? 2 * kGroup * 4 : 0)));
                    }
                    __syncwarp();
                    if constexpr (kF16) {
                        if (page >= 0) {
                            const int64_t at = a.kv.page_base(page, head) + ((j0 + kGroup * lane) & in_page);
                            bulk::load(raw_smem + land * C::kRawTile + lane * kGroupBytes,
                                       (kv ? a.kv.v : a.kv.k) + at * HD, kGroupBytes, &ctl.landed[land]);
                            if (kv == 0) {
                                bulk::load(&ctl.kscale[blocks % kRing][kGroup * lane], a.kv.k_scale + at, kGroup * 4, &ctl.landed[land]);
                                bulk::load(&ctl.vscale[blocks % kRing][kGroup * lane], a.kv.v_scale + at, kGroup * 4, &ctl.landed[land]);
                            }
                        }
                    } else {
                        constexpr int kHalves = HD / 64;
                        const int g = lane / kHalves, h = lane % kHalves;
                        const int pg = __shfl_sync(0xffffffffu, page, g & 7);
                        if (g < kU / kGroup && pg >= 0) {
                            const int64_t at = a.kv.page_base(pg, head) + ((j0 + kGroup * g) & in_page);
                            tma_load_2d(smem_addr(st_smem + land * C::kTile) + h * 16384 + g * (kGroup * 128),
                                        kv ? &v_map : &k_map, h * 64, (int)at, &ctl.landed[land]);
                        }
                    }
                }
            }
            if (!ok) break;
        }
        // an abort leaves copies in flight: they get a millisecond before shared memory goes
        if (!ok) {
            const uint64_t t0 = bulk::globaltimer_ns();
            while (bulk::globaltimer_ns() - t0 < 1000000ull) {}
        }
    } else if (wg == 2) {
        // ================= finishing tiles ===================================================
        uint32_t idx = 0, blocks = 0;
        bool ok = true;
        while (next(ok)) {
            for (int blk = it.blk0; ok && blk < it.blk1; blk++, blocks++) {
                const int j0 = blk * kU, slot = blocks % kRing;
                const int page = page_of(it.seq, it.k1, j0);
                if (wt < kU / kGroup && page < 0 && j0 + kGroup * lane < it.k1 &&
                    j0 + kGroup * lane + kGroup > it.k0)
                    flag(a.err, LAI_DEVERR_PAGE);
                const uint32_t groups = __ballot_sync(0xffffffffu, page >= 0);
                const bool whole = groups == 0xff && j0 >= it.k0 && j0 + kU <= it.k1;
                const bool mixed = paged::mixed(it, a.window, j0, kU);
                auto there = [&](int r) {
                    return j0 + r >= it.k0 && j0 + r < it.k1 && (groups >> (r / kGroup) & 1);
                };
                for (int kv = 0; kv < 2; kv++, idx++) {
                    const uint32_t land = idx % LD;
                    if (!(ok = wait(&ctl.landed[land], (idx / LD) & 1))) break;
                    if (kF16 && idx >= (uint32_t)ST && !(ok = wait(&ctl.empty[idx % ST], (idx / ST - 1) & 1))) break;
                    if (kv == 0) {  // the block's ring entries are free by now
                        if (kF16) {
                            const float vs = there(wt) ? ctl.vscale[slot][kF16 ? wt : 0] : 0.f;
                            const uint32_t u = __float_as_uint(vs) & 0x7fffffffu;
                            const bool fine = u < 0x7f800000u;
                            if (!whole || mixed) {  // weight 0 times a scale has to be 0
                                ctl.vscale[slot][kF16 ? wt : 0] = mixed && !fine ? 0.f : vs;
                                if (mixed && !fine) ctl.vbad[slot] = (int)blocks;
                            }
                            const uint32_t top = __reduce_max_sync(0xffffffffu, fine ? u : 0u);
                            const uint32_t low = __reduce_min_sync(0xffffffffu, fine && u ? u : 0x7f800000u);
                            if (lane == 0) ctl.vspan[slot][wt >> 5] = (top >> 23) << 16 | (255u - (low >> 23));
                        }
                        if (wt == 0) ctl.groups[slot] = (int)groups;
                        __syncwarp();
                        if (lane == 0) bulk::mbar_arrive(&ctl.info[slot]);
                    }
                    const uint32_t dst = smem_addr(st_smem + (idx % ST) * C::kTile);
                    bool bad = false, wrote = kF16;
                    if constexpr (kF16) {
                        constexpr int kIn = HD / 16, kAtOnce = 128 / kIn;  // runs of a row, rows at a time
                        const int c = wt % kIn, r_in = wt / kIn;
                        // a row's 8 lanes write 8 different 16-byte columns of a 128-byte line
                        const bool swap = HD == 128 && c >= kIn / 2;
                        const uint32_t src = smem_addr(raw_smem + land * C::kRawTile) + wt * 16;
#pragma unroll 4
                        for (int p = 0; p < 128 / kAtOnce; p++) {
                            const int r = p * kAtOnce + r_in;
                            uint4 raw = ld_shared16(src + p * 2048);
                            if (!whole && kv && !there(r)) raw = make_uint4(0, 0, 0, 0);
                            uint4 lo = make_uint4(half2_of<FMT, false>(raw.x), half2_of<FMT, true>(raw.x),
                                                  half2_of<FMT, false>(raw.y), half2_of<FMT, true>(raw.y));
                            uint4 hi = make_uint4(half2_of<FMT, false>(raw.z), half2_of<FMT, true>(raw.z),
                                                  half2_of<FMT, false>(raw.w), half2_of<FMT, true>(raw.w));
                            if (FMT == LAI_KV_E4M3 && mixed && kv) {
                                bad |= drop_nonfinite<true>(lo.x) | drop_nonfinite<true>(lo.y) |
                                       drop_nonfinite<true>(lo.z) | drop_nonfinite<true>(lo.w);
                                bad |= drop_nonfinite<true>(hi.x) | drop_nonfinite<true>(hi.y) |
                                       drop_nonfinite<true>(hi.z) | drop_nonfinite<true>(hi.w);
                            }
                            st_shared16(dst + chunk_off(r, 2 * c + swap), swap ? hi : lo);
                            st_shared16(dst + chunk_off(r, 2 * c + !swap), swap ? lo : hi);
                        }
                    } else if (kv && (!whole || mixed)) {  // thread = row of the tile
                        const bool gone = !there(wt);
                        if (gone || mixed) {
#pragma unroll 1
                            for (int c = 0; c < HD / 8; c++) {
                                const uint32_t at = dst + chunk_off(wt, c);
                                uint4 v = make_uint4(0, 0, 0, 0);
                                if (!gone) {
                                    v = ld_shared16(at);
                                    bad |= drop_nonfinite<false>(v.x) | drop_nonfinite<false>(v.y) |
                                           drop_nonfinite<false>(v.z) | drop_nonfinite<false>(v.w);
                                }
                                st_shared16(at, v);
                            }
                        }
                        wrote = true;
                    }
                    if (bad) ctl.vbad[slot] = (int)blocks;
                    if (wrote) bulk::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        bulk::mbar_arrive(&ctl.full[idx % ST]);
                        if (kF16) bulk::mbar_arrive(&ctl.taken[land]);
                    }
                }
            }
        }
    } else if (warp == 12) {
        // ================= MMAs ==============================================================
        constexpr uint32_t kIdS = idesc<kF16, 128, false>(), kIdO = idesc<kF16, HD, true>();
        const bool leader = elect_one();
        uint32_t idx = 0, n_q[2] = {0, 0}, n_mt[2] = {0, 0};
        bool ok = true;
        // what the leader issued so far arrives on bar when it is done
        auto commit = [&](uint64_t *bar) {
            if (leader) umma::commit(bar);
            __syncwarp();
        };
        auto scores = [&](int mt, uint32_t i) {
            const uint64_t kd = desc_kmajor(smem_addr(st_smem + (i % ST) * C::kTile));
            const uint64_t qd = desc_kmajor(smem_addr(q_smem) + mt * C::kTile);
            if (leader) {
#pragma unroll
                for (int t = kTerms - 1; t >= 0; t--)
#pragma unroll
                    for (int k = 0; k < HD / 16; k++) {
                        constexpr uint32_t kT = MT * C::kTile;
                        const uint32_t off = (k / 4) * 16384 + (k % 4) * 32;
                        mma_ss(tmem + mt * 128, qd + ((t * kT + off) >> 4), kd + (off >> 4), kIdS,
                               t != kTerms - 1 || k);
                    }
            }
            commit(&ctl.s_full[mt]);
        };
        while (next(ok)) {
            const int tiles = MT == 2 && it.rows > 128 ? 2 : 1;
            const int nb = it.blk1 - it.blk0;
            ok = wait(&ctl.full[idx % ST], (idx / ST) & 1);
            for (int mt = 0; ok && mt < tiles; mt++) {
                ok = wait(&ctl.q_full[mt], n_q[mt]++ & 1);
                umma::fence_after_sync();
                if (ok) scores(mt, idx);
            }
            if (!ok) break;
            commit(&ctl.empty[idx % ST]);
            for (int b = 0; ok && b < nb; b++) {
                const uint32_t vi = idx + 1, ki = idx + 2;
                const bool more = b + 1 < nb;
                for (int mt = 0; ok && mt < tiles; mt++) {
                    const uint64_t vd = desc_mnmajor(smem_addr(st_smem + (vi % ST) * C::kTile));
                    // keys 64 h .. of the block, once their weights are there
                    auto values = [&](int h) {
                        if (leader) {
#pragma unroll
                            for (int t = kTerms - 1; t >= 0; t--)
#pragma unroll
                                for (int k = 0; k < kU / 32; k++)
                                    mma_ts(tmem + kPV + mt * 128, tmem + kP + mt * 128 + t * 64 + (h * 4 + k) * 8,
                                           vd + (((h * 4 + k) * 2048) >> 4), kIdO,
                                           (MT == 2 && b > 0) || h || t != kTerms - 1 || k);
                        }
                        __syncwarp();
                    };
                    const uint32_t parity = n_mt[mt]++ & 1;
                    if (!(ok = wait(&ctl.p_full[mt][0], parity))) break;
                    if (!(ok = wait(&ctl.full[vi % ST], (vi / ST) & 1))) break;
                    umma::fence_after_sync();
                    values(0);
                    if (!(ok = wait(&ctl.p_full[mt][1], parity))) break;
                    umma::fence_after_sync();
                    if (MT == 1 && more) {  // the next scores before the rest of P V
                        if (!(ok = wait(&ctl.full[ki % ST], (ki / ST) & 1))) break;
                        umma::fence_after_sync();
                        scores(mt, ki);
                    }
                    values(1);
                    if (MT == 1 || !more) commit(&ctl.pv_full[mt]);
                    if (MT == 2 && more) {
                        if (!(ok = wait(&ctl.full[ki % ST], (ki / ST) & 1))) break;
                        umma::fence_after_sync();
                        scores(mt, ki);
                    }
                }
                if (!ok) break;
                commit(&ctl.empty[vi % ST]);
                if (more) commit(&ctl.empty[ki % ST]);
                idx += 2;
            }
        }
        // Every MMA is done before TMEM is given back: each result was waited for. After an abort
        // nobody waits, so the MMAs in flight get a millisecond.
        if (!ok) {
            const uint64_t t0 = bulk::globaltimer_ns();
            while (bulk::globaltimer_ns() - t0 < 1000000ull) {}
        }
    } else if (wg < 2) {
        // ================= softmax: a thread per row, or two =================================
        // Two tiles: warpgroup = tile. One tile: warpgroup `half` has keys 64 half .. of a block and
        // columns HD / 2 half .. of the output.
        constexpr bool kSplit = MT == 1;
        constexpr int kCols = kSplit ? HD / 2 : HD;
        const int mt = kSplit ? 0 : wg, half = kSplit ? wg : 0;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + lane_base + mt * 128, t_p = t_s + kP, t_pv = tmem + lane_base + kPV + mt * 128 + half * kCols;
        uint32_t n = 0, blocks = 0, n_group = 0, n_last = 0;  // this tile's blocks, all blocks, joins, last P Vs
        bool ok = true;
        auto join = [&]() {  // all that work on the tile, within the bound
            bulk::mbar_arrive(&ctl.group[mt]);
            return wait(&ctl.group[mt], n_group++ & 1);
        };
        // the other half's value of this row
        auto exchange = [&](float x, float &other) -> bool {
            float (*buf)[QF32 ? 128 : 1] = ctl.swap[QF32 ? n_group & 1 : 0];
            buf[half][QF32 ? wt : 0] = x;
            if (!(ok = join())) return false;
            other = buf[1 - half][QF32 ? wt : 0];
            return true;
        };
        while (next(ok)) {
            const int nb = it.blk1 - it.blk0;
            if (it.rows <= mt * 128) {  // no rows of this tile
                blocks += nb;
                continue;
            }
            const int head = it.head;
            const int r = mt * 128 + wt, fr = it.row0 + r, tok = a.by_group.of(fr);
            const int row_pos = it.pos0 + tok;  // of a row behind the last: not stored
            const int row_from = a.window ? row_pos - a.window : -1;  // sees (row_from, row_pos]
            // Q into shared memory, the warp's own 32 rows; the last scores of the item before are
            // done. kLanes lanes take a row, so that a load reads whole lines.
            const uint32_t my_rows = smem_addr(q_smem) + mt * C::kTile;  // this tile of the first term
            const int wrow = (warp & 3) * 32;                            // the warp's first row of it
            constexpr int kElem = QF32 ? 4 : 2, kLanes = HD * kElem / 16, kAtOnce = 32 / kLanes;
            const int run = lane % kLanes, sub = lane / kLanes;
            // rows of the warp as token and head of the group, counting up by `step`
            int tk, gh, step_t, step_g;
            auto first_row = [&](int from, int step) {
                step_t = a.by_group.of(step);
                step_g = step - step_t * a.group;
                const int f = it.row0 + mt * 128 + wrow + from;
                tk = a.by_group.of(f);
                gh = f - tk * a.group;
            };
            auto next_row = [&]() {
                tk += step_t;
                gh += step_g;
                if (gh >= a.group) gh -= a.group, tk++;
            };
            float c = a.scale_log2;
            {
                constexpr int kBatch = 32 / kAtOnce < 16 ? 32 / kAtOnce : 16;  // loads under way per lane
                const char *src = static_cast<const char *>(qp) +
                                  ((int64_t)it.q_row0 * a.ld_q + (int64_t)head * a.group * HD) * kElem + run * 16;
                first_row(sub, kAtOnce);
#pragma unroll 1
                for (int p0 = 0; p0 < 32 / kAtOnce; p0 += kBatch) {
                    uint4 raw[kBatch];
#pragma unroll
                    for (int p = 0; p < kBatch; p++) {
                        const int rr = (p0 + p) * kAtOnce + sub;
                        raw[p] = make_uint4(0, 0, 0, 0);
                        if (mt * 128 + wrow + rr < it.rows)
                            raw[p] = __ldg(reinterpret_cast<const uint4 *>(src + (tk * a.ld_q + gh * HD) * kElem));
                        next_row();
                    }
                    // (the other half has stored what it staged in these tiles)
                    if (kSplit && p0 == 0 && !(ok = join())) break;
#pragma unroll
                    for (int p = 0; p < kBatch; p++) {
                        const int rr = (p0 + p) * kAtOnce + sub;
                        float up = 1.f;
                        if (kF16) {  // the row's largest into [2^13, 2^14)
                            const uint32_t w[4] = {raw[p].x, raw[p].y, raw[p].z, raw[p].w};
                            uint32_t top = 0;
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                if (QF32) top = max(top, w[e] & 0x7fffffffu);
                                else top = max(top, max(w[e] << 16 & 0x7fffffffu, w[e] & 0x7fff0000u));
                            }
#pragma unroll
                            for (int o = kLanes / 2; o > 0; o >>= 1)
                                top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                            const int e = max((int)(top >> 23) - 127, -113);  // both powers are normal
                            up = pow2i(13 - e);
                            // the thread that owns the row keeps the other side of the scaling
                            const int mine = __shfl_sync(0xffffffffu, e, lane % kAtOnce * kLanes);
                            if (lane / kAtOnce == p0 + p) c = a.scale_log2 * pow2i(mine - 13);
                        }
                        // (each half has seen all rows' maxima, and writes half of the rows)
                        if (kSplit && ((p0 + p) * kAtOnce >= 16) != (half == 1)) continue;
                        if constexpr (QF32) {  // 4 values: half a 16-byte run of every term
                            float x[4] = {__uint_as_float(raw[p].x), __uint_as_float(raw[p].y),
                                          __uint_as_float(raw[p].z), __uint_as_float(raw[p].w)};
#pragma unroll
                            for (int e = 0; e < 4; e++) x[e] *= up;
#pragma unroll
                            for (int t = 0; t < kTerms; t++) {
                                const uint32_t lo = take2<kF16>(x[0], x[1]), hi = take2<kF16>(x[2], x[3]);
                                asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(
                                                 my_rows + t * MT * C::kTile + chunk_off(wrow + rr, run / 2) + run % 2 * 8),
                                             "r"(lo), "r"(hi)
                                             : "memory");
                            }
                        } else {
                            uint4 v = raw[p];
                            if (kF16) {
                                float x[8];
                                unpack<uint16_t>(v, x);
#pragma unroll
                                for (int e = 0; e < 8; e++) x[e] *= up;
                                v.x = pack2<true>(x[0], x[1]);
                                v.y = pack2<true>(x[2], x[3]);
                                v.z = pack2<true>(x[4], x[5]);
                                v.w = pack2<true>(x[6], x[7]);
                            }
                            st_shared16(my_rows + chunk_off(wrow + rr, run), v);
                        }
                    }
                }
                if (!ok) break;
                c = fmaxf(c, 1e-44f);  // masked scores, -inf, stay -inf
                bulk::fence_proxy_async_smem();
                bulk::mbar_arrive(&ctl.q_full[mt]);
            }
            // Weights are 2^(score - off); l and O are sums of these. off is the largest score, or, of an 8-bit
            // cache, the largest score plus exponent of the value's scale, less kLift.
            float off = neg_inf(), l = 0.f, alpha = 0.f;
            bool bad = false;
            constexpr int kKeep = kSplit ? kCols : 1;
            float o[kKeep];
#pragma unroll
            for (int d = 0; d < kKeep; d++) o[d] = 0.f;
            auto saw_bad = [&](uint32_t block) {
                bad |= *(volatile int *)&ctl.vbad[block % kRing] == (int)block;
            };
            auto add_pv = [&]() {
                umma::fence_after_sync();
#pragma unroll
                for (int g = 0; g < kKeep / 32; g++) {
                    uint32_t x[32];
                    umma::tmem_ld_32x32b_x32(t_pv + 32 * g, x);
                    umma::tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        o[(32 * g + i) % kKeep] = fmaf(o[(32 * g + i) % kKeep], alpha, __uint_as_float(x[i]));
                }
                umma::fence_before_sync();
            };
            for (int b = 0; b < nb; b++, n++, blocks++) {
                const int j0 = (it.blk0 + b) * kU, slot = blocks % kRing;
                if (!(ok = wait(&ctl.info[slot], (blocks / kRing) & 1) && wait(&ctl.s_full[mt], n & 1))) break;
                umma::fence_after_sync();
                if (MT == 2 && b > 0) saw_bad(blocks - 1);  // its P V came before these scores
                const int groups = ctl.groups[slot];
                const bool masked = groups != 0xff || j0 + kU - 1 > it.first || it.k0 > j0 ||
                                    (a.window && j0 <= it.last - a.window);
                // the row sees keys j0 + lo .. j0 + hi, as bits of 32 keys
                const int hi = row_pos - j0, lo = row_from + 1 - j0;
                auto seen = [&](int g) -> uint32_t {
                    const int h = min(max(hi + 1 - 32 * g, 0), 32), l = min(max(lo - 32 * g, 0), 32);
                    const uint32_t below_h = h == 32 ? 0xffffffffu : (1u << h) - 1;
                    const uint32_t below_l = l == 32 ? 0xffffffffu : (1u << l) - 1;
                    const uint32_t real = (groups >> (2 * g) & 1 ? 0xffffu : 0u) | (groups >> (2 * g + 1) & 1 ? 0xffff0000u : 0u);
                    return below_h & ~below_l & real;
                };
                const float4 *k4 = reinterpret_cast<const float4 *>(ctl.kscale[slot]);
                const float4 *v4 = reinterpret_cast<const float4 *>(ctl.vscale[slot]);
                bool each = false;  // the scales lie apart (the same for all warps)
                float ve = 0.f;
                if (kF16) {
                    const uint32_t *s4 = ctl.vspan[slot];
                    const uint32_t span = __vmaxu2(__vmaxu2(s4[0], s4[1]), __vmaxu2(s4[2], s4[3]));
                    const int e = (int)(span >> 16);
                    each = e + (int)(span & 255u) > 255 + kSpread;
                    ve = (float)min(max(e - 127, kLowScale), kTopScale);
                }
                // the largest score (below top) plus exponent of the value's scale, of the keys from j1 to j2;
                // rarely called, so short: S is read again
                auto exponents = [&](int j1, int j2, float top) {
                    float most = neg_inf();
#pragma unroll 1
                    for (int j = j1; j < j2; j += 16) {
                        uint32_t y[16];
                        umma::tmem_ld_32x32b_x16(t_s + j, y);
                        umma::tmem_wait_ld();
                        const uint32_t see = seen(j >> 5) >> (j & 16);
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const int u = __float_as_int(ctl.vscale[slot][kF16 ? j + i : 0]);
                            const float x = __uint_as_float(y[i]) * ctl.kscale[slot][kF16 ? j + i : 0];
                            const float e = (float)min(max((u >> 23 & 255) - 127, kLowScale), kTopScale);
                            most = fmaxf(most, see >> i & 1 ? __fmul_rn(x, c) - top + e : neg_inf());
                        }
                    }
                    return most;
                };
                // 32 scores with their keys' scales, masked; the maximum so far
                auto scale32 = [&](int g, float2 *x, float &top, auto mask) {
                    const uint32_t see = decltype(mask)::value ? seen(g) : 0u;
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        if (kF16) {
                            const float4 ks = k4[kF16 ? 8 * g + i / 2 : 0];
                            x[i] = __fmul2_rn(x[i], make_float2(ks.x, ks.y));
                            x[i + 1] = __fmul2_rn(x[i + 1], make_float2(ks.z, ks.w));
                        }
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            if (decltype(mask)::value) {
                                x[i + h].x = see >> (2 * (i + h)) & 1 ? x[i + h].x : neg_inf();
                                x[i + h].y = see >> (2 * (i + h) + 1) & 1 ? x[i + h].y : neg_inf();
                            }
                            top = max3(top, x[i + h].x, x[i + h].y);
                        }
                    }
                };
                // weights of 32 keys, into P
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                const float2 c2 = make_float2(c, c);
                auto weigh = [&](int g, const float2 *x, float base, auto mask) {
                    uint32_t w[kTerms][16];
                    const float2 nb2 = make_float2(-base, -base);
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        float4 vs = make_float4(1.f, 1.f, 1.f, 1.f);
                        if (kF16) vs = v4[kF16 ? 8 * g + i / 2 : 0];
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            // (the packed product and sum would become one fused operation)
                            float2 p = decltype(mask)::value
                                           ? make_float2(__fsub_rn(__fmul_rn(x[i + h].x, c), base),
                                                         __fsub_rn(__fmul_rn(x[i + h].y, c), base))
                                           : __ffma2_rn(x[i + h], c2, nb2);
                            // (scores of 2^20 and more are rounded before the subtraction, as the
                            // maximum was)
                            p = make_float2(ex2(p.x), ex2(p.y));
                            sum[h] = __fadd2_rn(sum[h], p);
                            if (kF16) p = __fmul2_rn(p, h ? make_float2(vs.z, vs.w) : make_float2(vs.x, vs.y));
#pragma unroll
                            for (int t = 0; t < kTerms; t++) w[t][i + h] = take2<kF16>(p.x, p.y);
                        }
                    }
#pragma unroll
                    for (int t = 0; t < kTerms; t++) tmem_st_x16(t_p + t * 64 + 16 * g, w[t]);
                    if (g & 1) {  // 64 keys' weights are there
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                        umma::fence_before_sync();
                        bulk::mbar_arrive(&ctl.p_full[mt][g >> 1]);
                    }
                };
                auto fetch = [&](int g, float2 *x) {  // without waiting
                    umma::tmem_ld_32x32b_x32(t_s + 32 * g, *reinterpret_cast<uint32_t (*)[32]>(x));
                };
                auto is_big = [&](float top) { return __any_sync(0xffffffffu, fabsf(top) > 1048576.f); };
                // moves off to the block's maximum; what l and O must be multiplied with
                auto move = [&](float top, float e, float slack) -> float {
                    // an infinite or NaN score: no weight of this row means anything any more
                    if (!(top < __int_as_float(0x7f800000))) l = __int_as_float(0x7fffffff);
                    // rounded up where scores are large, so that weights stay below 2^15; from 2^28 on
                    // their last place passes 2^kLift
                    const float to = kF16 && fabsf(top) < 268435456.f ? __fadd_ru(top, e - C::kLift) : top;
                    const float d = to - off;
                    if (!(d > slack)) return 1.f;  // (no key yet and none now: NaN)
                    off = to;
                    const float f = ex2(-d);  // off = -inf: 0
                    l *= f;
                    return f;
                };
                if constexpr (MT == 2) {
                    float2 x[kU / 2];
#pragma unroll
                    for (int g = 0; g < 4; g++) fetch(g, x + 16 * g);
                    umma::tmem_wait_ld();
                    float part[4] = {neg_inf(), neg_inf(), neg_inf(), neg_inf()};
                    auto scale_all = [&](auto mask) {
#pragma unroll
                        for (int g = 0; g < 4; g++) scale32(g, x + 16 * g, part[g], mask);
                    };
                    if (masked) scale_all(Yes{}); else scale_all(No{});
                    float top = max3(max3(part[0], part[1], part[2]), part[3], part[3]);
                    if (top != neg_inf()) top *= c;
                    if (each) ve = exponents(0, kU, top);
                    const float f = move(top, ve, kGrow);
                    if (b > 0 && __any_sync(0xffffffffu, f != 1.f)) {
                        // the scores' MMAs came after the last P V, so O is complete
#pragma unroll 1
                        for (int g = 0; g < HD / 16; g++) {
                            uint32_t y[16];
                            umma::tmem_ld_32x32b_x16(t_pv + 16 * g, y);
                            umma::tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; i++) y[i] = __float_as_uint(__uint_as_float(y[i]) * f);
                            tmem_st_x16(t_pv + 16 * g, y);
                        }
                    }
                    const float base = off == neg_inf() ? 0.f : off;
                    auto weigh_all = [&](auto mask) {
#pragma unroll
                        for (int g = 0; g < 4; g++) weigh(g, x + 16 * g, base, mask);
                    };
                    if (masked || is_big(top)) weigh_all(Yes{}); else weigh_all(No{});
                } else {
                    float2 x[kU / 4];  // this half's keys
                    fetch(2 * half, x);
                    fetch(2 * half + 1, x + 16);
                    umma::tmem_wait_ld();
                    float top = neg_inf(), other;
                    auto scale_half = [&](auto mask) {
#pragma unroll
                        for (int g = 0; g < 2; g++) scale32(2 * half + g, x + 16 * g, top, mask);
                    };
                    if (masked) scale_half(Yes{}); else scale_half(No{});
                    if (!exchange(top, other)) break;
                    top = max3(top, other, other);
                    if (top != neg_inf()) top *= c;
                    if (each) {
                        ve = exponents(64 * half, 64 * half + 64, top);
                        if (!exchange(ve, other)) break;
                        ve = fmaxf(ve, other);
                    }
                    if (b > 0) {  // P V of the block before, while S waited
                        if (!(ok = wait(&ctl.pv_full[mt], (n - 1) & 1))) break;
                        saw_bad(blocks - 1);
                        add_pv();
                    }
                    alpha = move(top, ve, 0.f);
                    const float base = off == neg_inf() ? 0.f : off;
                    auto weigh_half = [&](auto mask) {
#pragma unroll
                        for (int g = 0; g < 2; g++) weigh(2 * half + g, x + 16 * g, base, mask);
                    };
                    if (masked || is_big(top)) weigh_half(Yes{}); else weigh_half(No{});
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            }
            if (!ok) break;
            // the last P V: one commit per item with two tiles, one per block with one
            if (!(ok = wait(&ctl.pv_full[mt], (MT == 2 ? n_last++ : n - 1) & 1))) break;
            umma::fence_after_sync();
            saw_bad(blocks - 1);
            if (MT == 1) add_pv();
            if constexpr (kSplit) {
                float other;
                if (!exchange(l, other)) break;
                l += other;
            }
            // 32 of this thread's columns, before the division (rolled where it may be: the code of
            // all roles shares the instruction cache)
            constexpr int kPieces = kSplit ? kCols / 32 : 1;
            auto piece = [&](int g, float (&x)[32]) {
                if constexpr (MT == 2) {
                    uint32_t u[32];
                    __syncwarp();
                    umma::tmem_ld_32x32b_x32(t_pv + 32 * g, u);
                    umma::tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i++) x[i] = __uint_as_float(u[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i++) x[i] = o[(32 * g + i) % kKeep];
                }
            };
            // Infinities and NaN that were taken out of blocks whose rows differ in what they see:
            // add(d, value) for each that this row sees.
            auto mend = [&](auto add) {
                for (int j = max(it.blk0 * kU, it.k0); j < min(it.blk1 * kU, it.k1); j++) {
                    if (!paged::mixed(it, a.window, j / kU * kU, kU) || j > row_pos || j <= row_from) continue;
                    const int page = __ldg(a.kv.pages + (int64_t)it.seq * a.kv.max_pages + (j >> a.kv.log_page));
                    if (page < 0 || page >= a.kv.n_pages) continue;
                    const int64_t at = a.kv.page_base(page, head) + (j & in_page);
                    const float vs = kF16 ? __ldg(a.kv.v_scale + at) : 1.f;
#pragma unroll 1
                    for (int d = half * kCols; d < half * kCols + kCols; d++) {
                        const float v = element<FMT>(a.kv.v, at * HD + d) * vs;
                        if ((__float_as_uint(v) & 0x7f800000u) == 0x7f800000u) add(d, v);
                    }
                }
            };
            // 32 columns of this thread's row into the warp's rows of the Q tile (the next item's Q
            // is not there yet), the second half's in the second term's tile: 2 HD bytes a row
            const uint32_t staged = my_rows + half * MT * C::kTile;
            auto stage = [&](int g, const float (&x)[32], float inv) {
                if (QF32) {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        st_shared16(staged + chunk_off(wt, 8 * g + i),
                                    make_uint4(__float_as_uint(x[4 * i] * inv), __float_as_uint(x[4 * i + 1] * inv),
                                               __float_as_uint(x[4 * i + 2] * inv), __float_as_uint(x[4 * i + 3] * inv)));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float y[8] = {x[8 * i] * inv, x[8 * i + 1] * inv, x[8 * i + 2] * inv, x[8 * i + 3] * inv,
                                            x[8 * i + 4] * inv, x[8 * i + 5] * inv, x[8 * i + 6] * inv, x[8 * i + 7] * inv};
                        st_shared16(staged + chunk_off(wt, 4 * g + i), pack<uint16_t>(y));
                    }
                }
            };
            auto store = [&]() {  // the warp's staged rows, in whole lines
                constexpr int kOut = HD / 8, kOutRows = 32 / kOut;  // lanes a row, rows at once
                const int oc = lane % kOut, from = lane / kOut;
                __syncwarp();
                char *dst = static_cast<char *>(out) +
                            ((int64_t)it.q_row0 * a.kv.n_kv + head) * a.group * (HD * kElem) + half * (HD * 2) + oc * 16;
                const int64_t tok_bytes = (int64_t)a.kv.n_kv * a.group * (HD * kElem);
                first_row(from, kOutRows);
#pragma unroll 4
                for (int p = 0; p < 32 / kOutRows; p++, next_row()) {
                    const int rr = p * kOutRows + from;
                    if (mt * 128 + wrow + rr >= it.rows) continue;
                    st_vec(dst + tk * tok_bytes + gh * (HD * kElem), ld_shared16(staged + chunk_off(wrow + rr, oc)));
                }
                __syncwarp();
            };
            // parts: [row] off, [row] sum, then [d / 4][row][4]
            constexpr int64_t kPart = (int64_t)R * (HD + 2);
            auto part = [&](int cc) { return a.parts + ((int64_t)cc * 2 + (cc == it.c0 ? 1 : 0)) * kPart; };
            float mu = 0.f;
            if (!it.whole) {
                float *pp = a.parts + ((int64_t)blockIdx.x * 2 + (it.begins ? 1 : 0)) * kPart;
                if (half == 0) {
                    pp[r] = off;
                    pp[R + r] = l;
                }
#pragma unroll kPieces
                for (int g = 0; g < kCols / 32; g++) {
                    float x[32];
                    piece(g, x);
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<float4 *>(pp + 2 * R + ((half * (kCols / 4) + 8 * g + i / 4) * R + r) * 4) =
                            make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
                }
                umma::fence_before_sync();
                if (bad) mend([&](int d, float v) { pp[2 * R + (d / 4 * R + r) * 4 + d % 4] += v; });
                __threadfence();
                if (!(ok = join())) break;
                if (wt == 0 && half == 0) ctl.last[mt] = atomicAdd(a.counters + it.c0 * MT + mt, 1) == it.c1 - it.c0;
                if (!(ok = join())) break;
                if (!*(volatile int *)&ctl.last[mt]) continue;
                __threadfence();
                if (wt == 0 && half == 0) a.counters[it.c0 * MT + mt] = 0;  // ready for the next call
                float top = neg_inf();
                for (int cc = it.c0; cc <= it.c1; cc++) top = fmaxf(top, __ldcg(part(cc) + r));
                mu = top == neg_inf() ? 0.f : top;
                l = 0.f;
                for (int cc = it.c0; cc <= it.c1; cc++)
                    l = fmaf(__ldcg(part(cc) + R + r), ex2(__ldcg(part(cc) + r) - mu), l);
            }
            const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll kPieces
            for (int g = 0; g < kCols / 32; g++) {
                float x[32];
                if (it.whole) {
                    piece(g, x);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i++) x[i] = 0.f;
#pragma unroll 4
                    for (int cc = it.c0; cc <= it.c1; cc++) {
                        const float *pc = part(cc);
                        const float f = ex2(__ldcg(pc + r) - mu);
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 v = __ldcg(reinterpret_cast<const float4 *>(pc + 2 * R + ((half * (kCols / 4) + 8 * g + i / 4) * R + r) * 4));
                            x[i] = fmaf(v.x, f, x[i]);
                            x[i + 1] = fmaf(v.y, f, x[i + 1]);
                            x[i + 2] = fmaf(v.z, f, x[i + 2]);
                            x[i + 3] = fmaf(v.w, f, x[i + 3]);
                        }
                    }
                }
                stage(g, x, inv);
            }
            umma::fence_before_sync();
            if (it.whole && bad)
                mend([&](int d, float v) {
                    if (QF32) {
                        float *p = reinterpret_cast<float *>(q_smem + half * MT * C::kTile + chunk_off(wt, d % (HD / 2) / 4) + d % 4 * 4);
                        *p += v;
                    } else {
                        uint16_t *p = reinterpret_cast<uint16_t *>(q_smem + mt * C::kTile + chunk_off(wt, d / 8) + d % 8 * 2);
                        *p = from_f<uint16_t>(to_f(*p) + v);
                    }
                });
            store();
        }
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    if (threadIdx.x == 0 && ctl.abort) flag(a.err, LAI_DEVERR_TIMEOUT);
    if (warp == 12) umma::tmem_dealloc(tmem, 512);
}

// The cache as rows of head_dim BF16 values, copied 16 rows x 64 columns at a time.
using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                 CUtensorMapFloatOOBfill);
EncodeTiled encode_fn() {
    static std::once_flag once;
    static EncodeTiled fn = nullptr;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiled>(p);
    });
    return fn;
}
bool row_map(CUtensorMap *m, unsigned char *base, int64_t rows, int hd) {
    const cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)hd * 2};
    const cuuint32_t box[2] = {64, kGroup}, es[2] = {1, 1};
    const EncodeTiled fn = encode_fn();
    return fn && fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, es,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, int FMT, bool QF32>
int launch_wide(void *out, const void *q, const AttnArgs &a, cudaStream_t st) {
    using C = Cfg<HD, FMT, QF32>;
    constexpr size_t kSmem = (size_t)(C::MT * C::kTerms + C::kStages) * C::kTile +
                             (size_t)C::kRaw * C::kRawTile + sizeof(Ctl<HD, FMT, QF32>);
    static_assert(kSmem <= 227 * 1024, "one CTA's shared memory");
    auto kern = paged_attn_wide_kernel<HD, FMT, QF32>;
    // the warpgroups' register shares (setmaxnreg) add up to what the block is launched with
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, kern) != cudaSuccess || fa.numRegs != 128) return LAI_ERR_CUDA;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem) != cudaSuccess)
        return LAI_ERR_CUDA;
    if (C::S::most_blocks(a.kv, a.group) > INT32_MAX) return LAI_ERR_RANGE;
    CUtensorMap maps[2] = {};
    if (FMT == LAI_KV_BF16) {
        const int64_t rows = (a.kv.n_pages * a.kv.n_kv) << a.kv.log_page;
        if (rows > INT32_MAX) return LAI_ERR_RANGE;  // 32-bit coordinates
        if (!row_map(&maps[0], a.kv.k, rows, HD) || !row_map(&maps[1], a.kv.v, rows, HD)) return LAI_ERR_CUDA;
    }
    launch_pdl(kern, dim3(kSMs), dim3(kThreads), kSmem, st, out, q, a, maps[0], maps[1]);
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
