// paged_attention.cu - attention of new tokens over the paged cache: the entry points, and the
// kernel for few query rows per sequence (decoding, drafted tokens).
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q . k_j - max)   over the keys a row sees
//
// (qwen_causal_attention in the reference, src/tts_native.c:576-578, 653-655.) With few rows the
// cost is reading K and V once: HBM bound, 2 head_dim bytes per key and kv head for an 8-bit
// cache. What stands in the way of that bound is arithmetic per key (group x 2 head_dim products,
// and the conversion of 8-bit values), so the products go through the tensor cores with keys and
// values in the operand layout of mma.m16n8k16, and every warp has its own keys, with no barrier
// in the loop. One warp of a CTA only copies: it follows the page tables and keeps a ring of
// chunks (a chunk is what a warp takes at a time) filled with bulk copies, across the ends of
// items, so the other seven neither compute addresses nor hold loads in registers. (With loads
// straight into registers 64 x 4096 INT8 keys took 143 us, bound by their latency at the 12 warps
// that fit, when this took 137.)
//   Measured, 64 sequences of 4096 keys, 16 heads of 128 on 8, one token each: BF16 keys 174 us with
// F32 q (6.15 TB/s, 0.95 of a copy's bandwidth) and 166 with BF16 q (6.5 TB/s, 1.00), so HBM; E4M3
// 109 and INT8 121 us (5.1 and 4.6 TB/s): the warps' latency over about 1000 instructions per 32 keys
// (a third of them conversions to binary16; issue slots 46% used at the 14 warps that registers
// allow), and the count of copies: 4 per chunk, 101 us on their own. V in 4 blocks apart, so that no
// banks conflict, took 7 copies and 165 us, in 2 blocks 145, scales by 16-byte copies of the lanes
// 145, each when the rest took 137. Short calls are latency: one sequence
// of 777 keys 10.6 us, of which finding the work 2.5, the first keys through a warp 4.7, leaving
// parts 1.6, joining them 1.7.
//   * The sums over head_dim and over keys do not depend on the order of their terms. A lane
//     takes 16-byte runs of K, and the query is loaded with the same permutation; a lane's n
//     columns of V are a 16-byte run too, and the output is written back with that permutation.
//   * An MMA has 16 rows and a tile has 8: rows 8-15 carry the second term of the first 8. F32
//     queries become hi + lo in binary16 (22 bits; the 8-bit formats are exact in binary16), or
//     three bfloat16 terms (24 bits) over a BF16 cache, and so do the weights p. With BF16
//     queries the second rows still make the weights exact to 16 bits or more. (One term of them
//     over the 8-bit formats was no faster: the compiler spilt registers, 143 us when two took 126.)
//   * Each block's P V starts from zero and is added to the F32 accumulators by the FMA that
//     rescales them, so a long sequence does not add up the MMA's truncated sums.
//   * 8-bit: a key's scale multiplies its score, a value's scale its weight. In binary16 these
//     products are held relative to the row's own largest so far (which 2^-ve brings to 2^13 .. 2^14),
//     so neither a value that another row sees nor a large one under a small weight costs a row
//     bits: what is below 2^-38 of its largest product is rounded.
#include "bulk_copy.cuh"
#include "paged_attention.cuh"

namespace lai {

namespace {

using namespace paged;

constexpr int kWarps = 7;     // that compute; one more copies
constexpr int kMath = kWarps * 32, kThreads = kMath + 32;
constexpr int kHalf = 4;      // sums that the warps join in
constexpr int kRows = 8;      // rows of a tile
constexpr int kCtasPerSm = 2;
constexpr int kMaxCtas = kSMs * kCtasPerSm;
constexpr int kCounters = 1024;  // ints at the front of the scratch

template <int FMT> __host__ __device__ constexpr int step_keys() { return FMT == LAI_KV_BF16 ? 16 : 32; }  // of a chunk
template <int FMT> __host__ __device__ constexpr int block_keys() { return kWarps * step_keys<FMT>(); }
constexpr uint64_t kWaitNs = 1000000000ull;
__host__ __device__ constexpr int part_floats(int hd) { return kRows * (hd + 2); }

// ---- operands ----------------------------------------------------------------------------------
template <bool F16> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <bool F16> __device__ __forceinline__ float2 unpack2(uint32_t p) {
    float2 f;
    if (F16)
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
            : "=f"(f.x), "=f"(f.y)
            : "r"(p));
    else
        f = make_float2(bf16_lo(p), bf16_hi(p));
    return f;
}
// x as a 16-bit pair, x becoming what is left of it.
template <bool F16> __device__ __forceinline__ uint32_t take2(float &x0, float &x1) {
    const uint32_t p = pack2<F16>(x0, x1);
    const float2 f = unpack2<F16>(p);
    x0 -= f.x;
    x1 -= f.y;
    return p;
}
// c (+)= a b; FIRST: c = a b, without zeros having to be moved into c.
template <bool F16, bool FIRST>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                    uint32_t a3, uint32_t b0, uint32_t b1) {
#define LAI_MMA(T)                                                                            \
    if (FIRST)                                                                                \
        asm("mma.sync.aligned.m16n8k16.row.col.f32." T "." T ".f32 "                          \
            "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"             \
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])                                  \
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));                \
    else                                                                                      \
        asm("mma.sync.aligned.m16n8k16.row.col.f32." T "." T ".f32 "                          \
            "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"                 \
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])                                  \
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1))
    if (F16) {
        LAI_MMA("f16");
    } else {
        LAI_MMA("bf16");
    }
#undef LAI_MMA
}
// Zero what is an infinity or NaN among the elements of a stored word; true if there was one.
template <int FMT> __device__ __forceinline__ bool drop_nonfinite(uint32_t &x) {
    uint32_t gone;
    if (FMT == LAI_KV_BF16) gone = __vcmpeq2(x & 0x7f807f80u, 0x7f807f80u);
    else gone = __vcmpeq4(x & 0x7f7f7f7fu, 0x7f7f7f7fu);  // E4M3: NaN alone
    x &= ~gone;
    return gone != 0;
}

// 16 or 8 bytes of shared memory by one instruction: none of them arrives apart from the others.
__device__ __forceinline__ uint4 slot_load16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint2 slot_load8(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float2 slot_scales(uint32_t at) {
    const uint2 v = slot_load8(at);
    return make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
}

// One stored element as F32, without its scale.
template <int FMT> __device__ __forceinline__ float element(const unsigned char *v, int64_t i) {
    if (FMT == LAI_KV_BF16) return to_f(reinterpret_cast<const uint16_t *>(v)[i]);
    if (FMT == LAI_KV_I8) return (float)reinterpret_cast<const int8_t *>(v)[i];
    return unpack2<true>(e4m3x2_to_f16x2(v[i])).x;
}

template <int FMT> using FewSched = Sched<kRows, block_keys<FMT>(), 0>;

// A chunk in shared memory: rows of K, rows of V, scales of K, scales of V.
template <int HD, int FMT>
struct Chunk {
    static constexpr int kKeys = step_keys<FMT>(), kRow = HD * Fmt<FMT>::kBytes;
    static constexpr int kV = kKeys * kRow, kScaleK = 2 * kV, kScaleV = kScaleK + kKeys * 4;
    static constexpr int kBytes = FMT == LAI_KV_BF16 ? kScaleK : kScaleV + kKeys * 4;
    static constexpr int kRing = 10;
};

template <int HD, int FMT>
struct Smem {
    alignas(128) unsigned char ring[Chunk<HD, FMT>::kRing][Chunk<HD, FMT>::kBytes];
    alignas(16) float o[kHalf][kRows][HD + 4];  // rows apart by 4 banks
    alignas(16) uint4 q[HD / 16][32];
    uint2 q3[FMT == LAI_KV_BF16 ? HD / 16 : 1][32];   // the third terms
    float m[kHalf][kRows], l[kHalf][kRows];
    uint64_t full[Chunk<HD, FMT>::kRing], empty[Chunk<HD, FMT>::kRing];
    uint32_t there[Chunk<HD, FMT>::kRing];            // 16-key groups of a chunk that have a page, as bits
    uint32_t id[Chunk<HD, FMT>::kRing];               // the chunk that a slot was given to last
    SchedSmem sched;
    SeqSmem seqs;
    int bad;          // the item (counted) that infinities or NaN were taken out of
    int last, abort;
};
__device__ __forceinline__ void math_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kMath) : "memory"); }

template <int HD, int FMT, bool QF32>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
paged_attn_few_kernel(void *out, const void *__restrict__ qp, const AttnArgs a) {
    constexpr bool kF16 = FMT != LAI_KV_BF16;
    constexpr bool kThird = QF32 && !kF16;           // a third bfloat16 term
    constexpr int kBytes = Fmt<FMT>::kBytes;
    constexpr int kStep = step_keys<FMT>(), U = block_keys<FMT>();
    constexpr int NB = kStep / 8, NK = kStep / 16;   // 8-key and 16-key groups of a warp's step
    constexpr int kChunks = HD * kBytes / 64;        // 16-byte runs of K per lane and key
    constexpr int kPerChunk = kF16 ? 4 : 2;          // k16 steps that a run feeds
    constexpr int KS = HD / 16;                      // k16 steps of a score
    constexpr int ND = HD / 8;                       // 8-column groups of the output
    constexpr int VW = HD * kBytes / 32;             // 32-bit words of V per lane and key
    constexpr int kLift = 13;                        // log2 of an 8-bit cache's largest products
    static_assert(kChunks * kPerChunk == KS, "a lane's runs cover its share of head_dim");

    using Ck = Chunk<HD, FMT>;
    constexpr int kRing = Ck::kRing;
    extern __shared__ __align__(128) unsigned char smem_bytes[];
    auto &sm = *reinterpret_cast<Smem<HD, FMT> *>(smem_bytes);
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    pdl_wait_prior();
    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        for (int i = 0; i < kRing; i++) {
            bulk::mbar_init(&sm.full[i], 1);
            bulk::mbar_init(&sm.empty[i], 1);
            sm.id[i] = 0xffffffffu;
        }
        sm.abort = 0;
        sm.bad = 0;
        bulk::fence_barrier_init();
    }
    const AttnArgs as = cache_seqs<kThreads>(a, sm.seqs);
    if (as.kv.n_seqs == 0) return;  // the whole grid
    const Range range = find_range<FewSched<FMT>, kThreads>(as, sm.sched);
    if (range.w0 >= range.w1) return;  // the whole CTA

    // Bounded wait of a warp. When one runs out the CTA goes on with whatever is there (every
    // access stays in bounds), no further wait takes time, and the caller gets the flag.
    auto give_up = [&]() {
        sm.abort = 1;
        flag(a.err, LAI_DEVERR_TIMEOUT);
    };
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (!bulk::mbar_try_wait(bar, parity)) {
            const uint64_t t0 = bulk::globaltimer_ns();
            while (!bulk::mbar_try_wait(bar, parity) && !*(volatile int *)&sm.abort)
                if (bulk::globaltimer_ns() - t0 > kWaitNs) give_up();
        }
        __syncwarp();
    };
    const int in_page = a.kv.page_size() - 1;
    Walk<FewSched<FMT>> it;
    it.start(as, range);
    uint32_t chunk0 = 0;  // chunks of the blocks before this one

    if (warp == kWarps) {
        // ---- copies: lane 2 c + kk (8-bit) or c (BF16) looks up the page of 16-key group kk of chunk c
        static_assert(kWarps * NK <= 32, "a lane per 16-key group of a block");
        while (it.next(as)) {
            const Tile &tl = it.tl;
            const int head = it.kv_head();
            const int32_t *table = a.kv.pages + (int64_t)tl.seq * a.kv.max_pages;
            for (int blk = it.blk0; blk < it.blk1; blk++, chunk0 += kWarps) {
                const int j = blk * U + 16 * lane;
                int page = -1;
                if (lane < kWarps * NK && j < tl.k1 && j + 16 > tl.k0) {
                    page = __ldg(table + (j >> a.kv.log_page));
                    if (page < 0 || page >= a.kv.n_pages) {
                        flag(a.err, LAI_DEVERR_PAGE);
                        page = -1;
                    }
                }
                const uint32_t real = __ballot_sync(0xffffffffu, page >= 0);
                const int64_t at = a.kv.page_base(page >= 0 ? page : 0, head) + (j & in_page);
                for (int c = 0; c < kWarps; c++) {
                    const uint32_t id = chunk0 + c, slot = id % kRing;
                    if (id >= (uint32_t)kRing) wait(&sm.empty[slot], (id / kRing - 1) & 1);
                    const uint32_t there = real >> (c * NK) & ((1u << NK) - 1);
                    if (lane == 0) {
                        sm.there[slot] = there;
                        *(volatile uint32_t *)&sm.id[slot] = id;
                        bulk::mbar_arrive_expect_tx(&sm.full[slot],
                                                    __popc(there) * (2 * 16 * Ck::kRow + (kF16 ? 2 * 16 * 4 : 0)));
                    }
                    __syncwarp();
                    // one copy for both groups of a chunk that lies in one page: copies cost time each
                    const bool one = NK == 2 && a.kv.log_page > 4 && there == 3u;
                    const int kk = lane % NK;
                    if (lane / NK == c && page >= 0 && !(one && kk)) {
                        unsigned char *to = sm.ring[slot];
                        const int n = one ? 32 : 16;
                        bulk::load(to + kk * 16 * Ck::kRow, a.kv.k + at * Ck::kRow, n * Ck::kRow, &sm.full[slot]);
                        if (kF16) bulk::load(to + Ck::kScaleK + kk * 64, a.kv.k_scale + at, n * 4, &sm.full[slot]);
                        bulk::load(to + Ck::kV + kk * 16 * Ck::kRow, a.kv.v + at * Ck::kRow, n * Ck::kRow, &sm.full[slot]);
                        if (kF16) bulk::load(to + Ck::kScaleV + kk * 64, a.kv.v_scale + at, n * 4, &sm.full[slot]);
                    }
                }
            }
        }
        if (sm.abort) {  // copies may be in flight: they get a millisecond before shared memory goes
            const uint64_t t0 = bulk::globaltimer_ns();
            while (bulk::globaltimer_ns() - t0 < 1000000ull) {}
        }
        return;
    }

    const int n_heads = a.kv.n_kv * a.group;
    const uint32_t zero = (uint32_t)a.kv.log_page >> 8;  // as only the host knows
    for (int n_it = 1; it.next(as); n_it++) {
        const Tile &tl = it.tl;
        const int head = it.kv_head(), blk0 = it.blk0, blk1 = it.blk1;

        // the query: lane (g, t) holds row g's elements 4 at a time, hi in the MMA's row g and
        // the rest of it in row g + 8
        float row_scale = a.scale_log2;
        const int row = tl.row0 + g, tok = a.by_group.of(row);
        const bool row_ok = g < tl.rows;
        const int row_pos = row_ok ? tl.pos0 + tok : -1;
        const int row_from = a.window ? row_pos - a.window : -1;  // sees keys in (row_from, row_pos]
        {
            const int64_t at = ((int64_t)tl.q_row0 + tok) * a.ld_q +
                               (int64_t)(head * a.group + (row - tok * a.group)) * HD;
            // the 4 elements that the lane needs in step s
            auto load4 = [&](int s, float (&x)[4]) {
                const int d = (s / kPerChunk * 4 + t) * (kPerChunk * 4) + s % kPerChunk * 4;
                x[0] = x[1] = x[2] = x[3] = 0.f;
                if (!row_ok) return;
                if (QF32) {
                    const float4 f = *reinterpret_cast<const float4 *>(static_cast<const float *>(qp) + at + d);
                    x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
                } else {
                    const uint2 f = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(qp) + at + d);
                    x[0] = bf16_lo(f.x); x[1] = bf16_hi(f.x); x[2] = bf16_lo(f.y); x[3] = bf16_hi(f.y);
                }
            };
            float up = 1.f;
            if (kF16) {  // the row's largest into [2^13, 2^14)
                uint32_t top = 0;
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    float x[4];
                    load4(s, x);
#pragma unroll
                    for (int e = 0; e < 4; e++) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
                }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int e = max((int)(top >> 23) - 127, -113);  // 2^(13 - e) and its reciprocal are normal
                up = pow2i(13 - e);
                row_scale *= pow2i(e - 13);
            }
#pragma unroll 1
            for (int s = warp; s < KS; s += kWarps) {  // the warp's share
                float x[4];
                load4(s, x);
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] *= up;
                uint4 v;
                v.x = take2<kF16>(x[0], x[1]);
                v.z = take2<kF16>(x[2], x[3]);
                v.y = QF32 ? take2<kF16>(x[0], x[1]) : 0u;
                v.w = QF32 ? take2<kF16>(x[2], x[3]) : 0u;
                sm.q[s][lane] = v;
                if constexpr (kThird) sm.q3[s][lane] = make_uint2(pack2<false>(x[0], x[1]), pack2<false>(x[2], x[3]));
            }
            math_sync();
        }

        // weights are 2^(score - m), m the maximum; l is their sum, o 2^-ve times the sum of their
        // products with the values
        float m = neg_inf(), l = 0.f, ve = 0.f, o[ND][2];
#pragma unroll
        for (int n = 0; n < ND; n++) o[n][0] = o[n][1] = 0.f;
        bool bad = false;

        for (int blk = blk0; blk < blk1; blk++, chunk0 += kWarps) {
            const int j0 = blk * U + warp * kStep;
            const uint32_t id = chunk0 + warp, slot = id % kRing;
            // A slot's chunks belong to different warps, and a parity only tells neighbouring phases
            // apart: a warp looks at its phase once the slot is its chunk's.
            if (*(volatile uint32_t *)&sm.id[slot] != id) {
                const uint64_t t0 = bulk::globaltimer_ns();
                while (*(volatile uint32_t *)&sm.id[slot] != id && !*(volatile int *)&sm.abort)
                    if (bulk::globaltimer_ns() - t0 > kWaitNs) give_up();
            }
            __syncwarp();
            wait(&sm.full[slot], (id / kRing) & 1);
            const uint32_t from = bulk::smem_addr(sm.ring[slot]);  // read by slot_load alone
            const uint32_t there = sm.there[slot];
            if (there == 0) {  // none of its keys
                __syncwarp();
                if (lane == 0) bulk::mbar_arrive(&sm.empty[slot]);
                continue;
            }
            const bool whole = there == (1u << NK) - 1 && j0 >= tl.k0 && j0 + kStep <= tl.k1;
            // ---- scores
            // (step by step over head_dim, so that the groups' MMAs stand between one group's)
            float cs[NB][4], sc[NB][2];
            uint4 kr[NB];
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const uint4 q = sm.q[s][lane];
                uint2 q3 = make_uint2(0u, 0u);
                if constexpr (kThird) q3 = sm.q3[s][lane];
#pragma unroll
                for (int n = 0; n < NB; n++) {
                    if (s % kPerChunk == 0)
                        kr[n] = slot_load16(from + (8 * n + g) * Ck::kRow + 16 * t + 64 * (s / kPerChunk));
                    const uint4 r = kr[n];
                    uint32_t b0, b1;
                    if constexpr (kF16) {
                        const int i = s % 4;
                        const uint32_t x = i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w;
                        b0 = half2_of<FMT, false>(x);
                        b1 = half2_of<FMT, true>(x);
                    } else {
                        b0 = s % 2 ? r.z : r.x;
                        b1 = s % 2 ? r.w : r.y;
                    }
                    if constexpr (kThird) {
                        if (s == 0) mma<kF16, true>(cs[n], q3.x, 0u, q3.y, 0u, b0, b1);
                        else mma<kF16, false>(cs[n], q3.x, 0u, q3.y, 0u, b0, b1);
                    }
                    if (s == 0 && !kThird) mma<kF16, true>(cs[n], q.x, q.y, q.z, q.w, b0, b1);
                    else mma<kF16, false>(cs[n], q.x, q.y, q.z, q.w, b0, b1);
                }
            }
#pragma unroll
            for (int n = 0; n < NB; n++) {
                sc[n][0] = cs[n][0] + cs[n][2];
                sc[n][1] = cs[n][1] + cs[n][3];
            }
            // ---- mask, running maximum
            float2 ks[NB], vs[NB];
            if (kF16) {
#pragma unroll
                for (int n = 0; n < NB; n++) {
                    ks[n] = slot_scales(from + Ck::kScaleK + (8 * n + 2 * t) * 4);
                    vs[n] = slot_scales(from + Ck::kScaleV + (8 * n + 2 * t) * 4);
                }
            }
            const bool uneven = mixed(tl, a.window, j0, kStep);
            const bool all = whole && !uneven;  // every row sees every key
            float top = neg_inf();
#pragma unroll
            for (int n = 0; n < NB; n++) {
                const float k0 = kF16 ? row_scale * ks[n].x : row_scale, k1 = kF16 ? row_scale * ks[n].y : row_scale;
                sc[n][0] *= k0;
                sc[n][1] *= k1;
            }
            if (!all) {
#pragma unroll
                for (int n = 0; n < NB; n++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int j = j0 + 8 * n + 2 * t + i;
                        const bool see = j <= row_pos && j > row_from && (there >> (n / 2) & 1);
                        sc[n][i] = see ? sc[n][i] : neg_inf();
                        if (kF16) {
                            float &f = i ? vs[n].y : vs[n].x;
                            f = see ? f : 0.f;
                        }
                    }
            }
#pragma unroll
            for (int n = 0; n < NB; n++) top = fmaxf(top, fmaxf(sc[n][0], sc[n][1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float mn = fmaxf(m, top);
            const float mu = mn == neg_inf() ? 0.f : mn;
            const float grown = m - mu;  // m = -inf: nothing to keep
            float alpha = ex2(grown);    // 1 where the maximum did not move, whatever its last place
            m = mn;
            // ---- weights
            float lsum = 0.f, ptop = 0.f, down = 1.f;
#pragma unroll
            for (int n = 0; n < NB; n++) {
                sc[n][0] = ex2(sc[n][0] - mu);
                sc[n][1] = ex2(sc[n][1] - mu);
                lsum += sc[n][0] + sc[n][1];
                if (kF16) {  // a masked value's scale is 0 by now
                    sc[n][0] *= vs[n].x;
                    sc[n][1] *= vs[n].y;
                    ptop = fmaxf(ptop, fmaxf(fabsf(sc[n][0]), fabsf(sc[n][1])));
                }
            }
            l = fmaf(l, alpha, lsum);
            if (kF16) {
                ptop = fmaxf(ptop, __shfl_xor_sync(0xffffffffu, ptop, 1));
                ptop = fmaxf(ptop, __shfl_xor_sync(0xffffffffu, ptop, 2));
                // the step's largest product, and that of what is kept, which falls as the maximum grows
                const int e = min(max((int)(__float_as_uint(ptop) >> 23) - 127 - kLift, -126), 114);
                const float now = fmaxf(ve + grown, (float)e);
                alpha = ex2(grown + (ve - now));
                down = ex2(-now);
                ve = now;
            }
            uint32_t pa[NK][kThird ? 6 : 4];
#pragma unroll
            for (int n = 0; n < NB; n++) {
                float p0 = sc[n][0] * down, p1 = sc[n][1] * down;
                uint32_t *pk = pa[n / 2] + (n & 1) * 2;
                pk[0] = take2<kF16>(p0, p1);
                if constexpr (kThird) {
                    pk[1] = take2<kF16>(p0, p1);
                    pa[n / 2][4 + (n & 1)] = pack2<false>(p0, p1);
                } else {
                    pk[1] = pack2<kF16>(p0, p1);
                }
            }
            // ---- values
            uint32_t vr[NK][4][VW];
#pragma unroll
            for (int kk = 0; kk < NK; kk++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t p = from + Ck::kV + (16 * kk + 2 * t + (i & 1) + 8 * (i >> 1)) * Ck::kRow;
                    if constexpr (VW == 2) {
                        const uint2 x = slot_load8(p + 8 * g);
                        vr[kk][i][0] = x.x; vr[kk][i][1] = x.y;
                    } else {
#pragma unroll
                        for (int c = 0; c < VW / 4; c++) {
                            const uint4 x = slot_load16(p + 16 * g + 128 * c);
                            vr[kk][i][4 * c] = x.x; vr[kk][i][4 * c + 1] = x.y;
                            vr[kk][i][4 * c + 2] = x.z; vr[kk][i][4 * c + 3] = x.w;
                        }
                    }
                }
            // What is not there may be anything, and weight 0 times it has to be 0. And a step whose
            // keys some rows of the tile see and others do not gives every row 0 x v for the keys it
            // must not see: infinities and NaN are taken out of such a step, and added to the rows
            // that see them at the end. (Of a part step whose rows all see the same keys nothing is
            // taken: what is there is seen.)
            if (!all) {
#pragma unroll
                for (int kk = 0; kk < NK; kk++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int j = j0 + 16 * kk + 2 * t + (i & 1) + 8 * (i >> 1);
                        const bool ok = (there >> kk & 1) && j >= tl.k0 && j < tl.k1;
#pragma unroll
                        for (int w = 0; w < VW; w++) {
                            uint32_t &x = vr[kk][i][w];
                            x = ok ? x : 0u;
                            if (FMT != LAI_KV_I8 && uneven) bad |= drop_nonfinite<FMT>(x);
                        }
                    }
            }
            auto column = [&](int n, uint32_t (&b0)[NK], uint32_t (&b1)[NK]) {
                float c[4];
#pragma unroll
                for (int kk = 0; kk < NK; kk++) {
                    const uint32_t *pk = pa[kk];
                    if constexpr (kThird) {
                        if (kk == 0) mma<kF16, true>(c, pk[4], 0u, pk[5], 0u, b0[kk], b1[kk]);
                        else mma<kF16, false>(c, pk[4], 0u, pk[5], 0u, b0[kk], b1[kk]);
                    }
                    if (kk == 0 && !kThird) mma<kF16, true>(c, pk[0], pk[1], pk[2], pk[3], b0[kk], b1[kk]);
                    else mma<kF16, false>(c, pk[0], pk[1], pk[2], pk[3], b0[kk], b1[kk]);
                }
                o[n][0] = fmaf(o[n][0], alpha, c[0] + c[2]);
                o[n][1] = fmaf(o[n][1], alpha, c[1] + c[3]);
            };
#pragma unroll
            for (int wd = 0; wd < VW; wd++) {
                uint32_t b0[NK], b1[NK];
                if constexpr (kF16) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {  // bytes 2h, 2h + 1 of the word
                        uint32_t x[NK], y[NK];
#pragma unroll
                        for (int kk = 0; kk < NK; kk++) {
                            x[kk] = prmt(vr[kk][0][wd], vr[kk][1][wd], h ? 0x7362 : 0x5140);
                            y[kk] = prmt(vr[kk][2][wd], vr[kk][3][wd], h ? 0x7362 : 0x5140);
                            b0[kk] = half2_of<FMT, false>(x[kk]);
                            b1[kk] = half2_of<FMT, false>(y[kk]);
                        }
                        column(4 * wd + 2 * h, b0, b1);
#pragma unroll
                        for (int kk = 0; kk < NK; kk++) {
                            b0[kk] = half2_of<FMT, true>(x[kk]);
                            b1[kk] = half2_of<FMT, true>(y[kk]);
                        }
                        column(4 * wd + 2 * h + 1, b0, b1);
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
#pragma unroll
                        for (int kk = 0; kk < NK; kk++) {
                            b0[kk] = prmt(vr[kk][0][wd], vr[kk][1][wd], h ? 0x7632 : 0x5410);
                            b1[kk] = prmt(vr[kk][2][wd], vr[kk][3][wd], h ? 0x7632 : 0x5410);
                        }
                        column(2 * wd + h, b0, b1);
                    }
                }
                if (wd == (VW == 8 ? 4 : 0)) {
                    // The slot's next copy writes through the async proxy, which an arrival's release
                    // does not keep behind generic loads still in flight: with no more than __syncwarp
                    // between loads and arrival, 0.4% of calls with many short BF16 sequences were
                    // wrong. So the arrival waits for products of every load (of all lanes: an MMA
                    // takes the whole warp's operands; of all bytes of a load: it is one instruction).
                    const float after = VW == 8 ? o[0][0] + o[ND / 2][0] : o[0][0];
                    if (lane == 0) bulk::mbar_arrive(&sm.empty[slot] + (__float_as_uint(after) & zero));
                }
            }
        }

        // ---- join the warps: the upper half's sums into the lower half's, those in shared memory
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (FMT != LAI_KV_I8 && bad) sm.bad = n_it;
        // Column 2t + i of group n: the lane that holds it took its V from the run of lanes with
        // g = 2t + i. Groups 4 k .. 4 k + 3 are neighbours in the output.
        auto run_of = [&](int k, int i) {
            const int gg = 2 * t + i, n = 4 * k;
            return VW == 2 ? gg * 8 + n : kF16 ? gg * 16 + n : (gg + 8 * (n / 8)) * 8 + n % 8;
        };
        const float unit = kF16 ? ex2(ve) : 1.f;
        const int half = warp % kHalf;
        if (warp >= kHalf) {
            if (t == 0) sm.m[half][g] = m, sm.l[half][g] = l;
#pragma unroll
            for (int k = 0; k < ND / 4; k++)
#pragma unroll
                for (int i = 0; i < 2; i++)
                    *reinterpret_cast<float4 *>(&sm.o[half][g][run_of(k, i)]) =
                        make_float4(o[4 * k][i] * unit, o[4 * k + 1][i] * unit, o[4 * k + 2][i] * unit, o[4 * k + 3][i] * unit);
        }
        math_sync();
        if (warp < kHalf) {
            const bool both = warp + kHalf < kWarps;
            const float mo = both ? sm.m[half][g] : neg_inf(), lo = both ? sm.l[half][g] : 0.f;
            const float mx = fmaxf(m, mo), mu = mx == neg_inf() ? 0.f : mx;
            const float ca = ex2(m - mu), cb = ex2(mo - mu), cu = ca * unit;
            __syncwarp();
            if (t == 0) {
                sm.l[half][g] = fmaf(lo, cb, l * ca);
                sm.m[half][g] = mx;
            }
#pragma unroll
            for (int k = 0; k < ND / 4; k++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    float4 *p = reinterpret_cast<float4 *>(&sm.o[half][g][run_of(k, i)]);
                    const float4 x = both ? *p : make_float4(0.f, 0.f, 0.f, 0.f);
                    *p = make_float4(fmaf(x.x, cb, o[4 * k][i] * cu), fmaf(x.y, cb, o[4 * k + 1][i] * cu),
                                     fmaf(x.z, cb, o[4 * k + 2][i] * cu), fmaf(x.w, cb, o[4 * k + 3][i] * cu));
                }
        }
        math_sync();
        // from here each of 128 threads owns kOwn columns of a row
        constexpr int kOwn = kRows * HD / 128;
        const int e = threadIdx.x * kOwn, r = e / HD, col = e % HD;
        const bool owner = threadIdx.x < 128;
        float acc[kOwn], sum, top;
        auto clear = [&]() {
#pragma unroll
            for (int i = 0; i < kOwn; i++) acc[i] = 0.f;
            sum = 0.f;
        };
        // adds the state (pm, pl, pv) of some keys; top is their common maximum by now
        auto add = [&](float pm, float pl, const float (&pv)[kOwn]) {
            const float f = ex2(pm - (top == neg_inf() ? 0.f : top));
            sum = fmaf(pl, f, sum);
#pragma unroll
            for (int i = 0; i < kOwn; i++) acc[i] = fmaf(pv[i], f, acc[i]);
        };
        auto write = [&]() {
            if (r >= tl.rows) return;
            const int fr = tl.row0 + r, tk = a.by_group.of(fr);
            const int64_t to = (((int64_t)tl.q_row0 + tk) * n_heads + head * a.group + (fr - tk * a.group)) * HD + col;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
            for (int i = 0; i < kOwn; i += 4)
                if (QF32)
                    *reinterpret_cast<float4 *>(static_cast<float *>(out) + to + i) =
                        make_float4(acc[i] * inv, acc[i + 1] * inv, acc[i + 2] * inv, acc[i + 3] * inv);
                else
                    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(out) + to + i) =
                        make_uint2(pack_bf16x2(acc[i] * inv, acc[i + 1] * inv), pack_bf16x2(acc[i + 2] * inv, acc[i + 3] * inv));
        };
        auto take4 = [](float (&to)[kOwn], int i, const float4 &x) {
            to[i] = x.x; to[i + 1] = x.y; to[i + 2] = x.z; to[i + 3] = x.w;
        };
        const bool alone = it.begins && it.ends;
        float *pp = a.parts + ((int64_t)blockIdx.x * 2 + (it.begins ? 1 : 0)) * part_floats(HD);
        if (owner) {
            clear();
            top = neg_inf();
#pragma unroll
            for (int x = 0; x < kHalf; x++) top = fmaxf(top, sm.m[x][r]);
#pragma unroll
            for (int x = 0; x < kHalf; x++) {
                float v[kOwn];
#pragma unroll
                for (int i = 0; i < kOwn; i += 4) take4(v, i, *reinterpret_cast<const float4 *>(&sm.o[x][r][col + i]));
                add(sm.m[x][r], sm.l[x][r], v);
            }
            if (FMT != LAI_KV_I8 && sm.bad == n_it && r < tl.rows) {
                const int p = tl.pos0 + a.by_group.of(tl.row0 + r);
                for (int j = max(blk0 * U, tl.k0); j < min(blk1 * U, tl.k1); j++) {
                    if (!mixed(tl, a.window, j / kStep * kStep, kStep) || j > p || (a.window && j <= p - a.window)) continue;
                    const int page = __ldg(a.kv.pages + (int64_t)tl.seq * a.kv.max_pages + (j >> a.kv.log_page));
                    if (page < 0 || page >= a.kv.n_pages) continue;
                    const int64_t at = (a.kv.page_base(page, head) + (j & in_page)) * HD + col;
#pragma unroll
                    for (int i = 0; i < kOwn; i++) {
                        const float v = element<FMT>(a.kv.v, at + i);
                        acc[i] += (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u ? v : 0.f;
                    }
                }
            }
            if (alone) {
                write();
                continue;
            }
            // parts: [row] max, [row] sum, [row][column]
            if (col == 0) {
                pp[r] = top;
                pp[kRows + r] = sum;
            }
#pragma unroll
            for (int i = 0; i < kOwn; i += 4)
                *reinterpret_cast<float4 *>(pp + 2 * kRows + e + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
        }
        if (alone) continue;
        const int c0 = range.cta_of(it.item0), c1 = range.cta_of(it.item1 - 1);
        math_sync();
        if (threadIdx.x == 0) {
            __threadfence();  // for the whole CTA, whose writes the barrier put before it
            const bool last = atomicAdd(a.counters + c0, 1) == c1 - c0;
            __threadfence();
            if (last) a.counters[c0] = 0;  // ready for the next call
            sm.last = last;
        }
        math_sync();
        if (!sm.last) continue;
        if (!owner) continue;
        // (More at once, or the parts dealt out to the warps, was not faster: a call's last CTA runs
        // this code for the first time, and its length counts.)
        constexpr int kAtOnce = 4;  // the parts in their order, so many of them under way
        clear();
        top = neg_inf();
#pragma unroll 1
        for (int first = c0; first <= c1; first += kAtOnce) {
            float pm[kAtOnce], pl[kAtOnce], pv[kAtOnce][kOwn];
#pragma unroll
            for (int c = 0; c < kAtOnce; c++) {
                const int ci = min(first + c, c1);  // (the first part is its CTA's second)
                const float *pc = a.parts + (ci * 2 + (ci == c0)) * part_floats(HD);
                pm[c] = __ldcg(pc + r);
                pl[c] = __ldcg(pc + kRows + r);
#pragma unroll
                for (int i = 0; i < kOwn; i += 4)
                    take4(pv[c], i, __ldcg(reinterpret_cast<const float4 *>(pc + 2 * kRows + e + i)));
            }
#pragma unroll
            for (int c = 1; c < kAtOnce; c++)
                if (first + c > c1) pm[c] = neg_inf(), pl[c] = 0.f;  // the last one again: weight 0
            const float was = top;
#pragma unroll
            for (int c = 0; c < kAtOnce; c++) top = fmaxf(top, pm[c]);
            const float f = ex2(was - (top == neg_inf() ? 0.f : top));
            sum *= f;
#pragma unroll
            for (int i = 0; i < kOwn; i++) acc[i] *= f;
#pragma unroll
            for (int c = 0; c < kAtOnce; c++) add(pm[c], pl[c], pv[c]);
        }
        write();
    }
}

template <int HD, int FMT, bool QF32>
int launch_few(void *out, const void *q, const AttnArgs &a, cudaStream_t st) {
    const int64_t most = FewSched<FMT>::most_blocks(a.kv, a.group);
    if (most > INT32_MAX) return LAI_ERR_RANGE;
    constexpr size_t kSmem = sizeof(Smem<HD, FMT>);
    static_assert(kSmem * kCtasPerSm <= 226 * 1024, "shared memory of an SM");
    auto kern = paged_attn_few_kernel<HD, FMT, QF32>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem) != cudaSuccess)
        return LAI_ERR_CUDA;
    launch_pdl(kern, dim3((unsigned)(most < kMaxCtas ? most : kMaxCtas)), dim3(kThreads), kSmem, st, out, q, a);
    return launch_status();
}

// Which kernel. The few-row one reads the keys once per 8 rows of a sequence, the wide one once per
// 128 or 256 but starts slowly and splits coarsely, so it wants several tiles of 8 in a sequence
// and enough of them in all. Measured over 1500 keys, 16 heads on 8, us (few / wide):
//   16 sequences: BF16 q, BF16 cache, 10 rows each 41 / 38, 24 rows 56 / 38; INT8 cache 16 rows
//   43 / 49, 24 rows 55 / 49; F32 q, BF16 cache 16 rows 45 / 57, 24 rows 60 / 58; INT8 cache
//   24 rows 49 / 57, 32 rows 62 / 57
//   4 sequences of 32 rows: 26 / 24 (BF16 q, BF16), 28 / 31 (F32 q); 1 of 64: 19 / 25, 20 / 28.
inline bool many_rows(int64_t rows, int n_seqs, int n_kv, bool f32, bool eight_bit) {
    const int64_t per_seq = 8 + (eight_bit ? 8 : 0) + (f32 ? 8 : 0);
    return rows > per_seq * n_seqs && rows / 8 * n_kv >= (f32 ? 256 : 128);
}

template <bool QF32>
int attention_entry(void *out, const void *q, int64_t ld_q, int64_t n_rows, int n_heads,
                    const lai_paged_kv_t *kv, const lai_paged_batch_t *b, float scale, int window,
                    void *scratch, int *err, lai_stream_t stream) {
    AttnArgs a;
    const int st = check(kv, b, n_rows, &a.kv);
    if (st != LAI_OK) return st;
    if (n_rows == 0 || b->n_seqs == 0) return LAI_OK;
    constexpr int kEsize = QF32 ? 4 : 2;
    if (!out || !q || !scratch || n_heads <= 0 || window < 0 || n_heads % kv->n_kv_heads != 0 ||
        n_heads / kv->n_kv_heads > 16)
        return LAI_ERR_INVALID;
    const int64_t width = (int64_t)n_heads * kv->head_dim;
    if (ld_q < width || ld_q % (16 / kEsize) != 0 || !aligned16(q) || !aligned16(out) ||
        !aligned16(scratch))
        return LAI_ERR_INVALID;
    if (n_rows * (n_heads / kv->n_kv_heads) + b->n_seqs >= 1 << 28) return LAI_ERR_RANGE;
    const size_t ob = paged::row_bytes(n_rows, width, width, kEsize);
    const size_t qb = paged::row_bytes(n_rows, ld_q, width, kEsize);
    const size_t wb = lai_paged_attention_scratch_bytes(kv->head_dim);
    if (overlaps(out, ob, q, qb) || hits_cache(kv, out, ob) || hits_cache(kv, scratch, wb) ||
        overlaps(scratch, wb, out, ob) || overlaps(scratch, wb, q, qb))
        return LAI_ERR_ALIAS;
    a.group = n_heads / kv->n_kv_heads;
    a.by_group = Div::by(a.group);
    a.window = window < (1 << 30) ? window : 0;  // positions are below 2^31: it masks nothing
    a.scale_log2 = scale * kLog2e;
    a.ld_q = ld_q;
    a.counters = static_cast<int *>(scratch);
    a.parts = reinterpret_cast<float *>(a.counters + kCounters);
    a.err = err;
    const cudaStream_t cs = as_stream(stream);
    if (many_rows(n_rows * a.group, b->n_seqs, kv->n_kv_heads, QF32, kv->format != LAI_KV_BF16) &&
        a.scale_log2 > 1e-30f)
        return attention_wide(out, q, QF32, kv->head_dim, kv->format, a, cs);
#define LAI_FEW(FMT)                                                             \
    (kv->head_dim == 128 ? launch_few<128, FMT, QF32>(out, q, a, cs) : launch_few<64, FMT, QF32>(out, q, a, cs))
    switch (kv->format) {
        case LAI_KV_BF16: return LAI_FEW(LAI_KV_BF16);
        case LAI_KV_E4M3: return LAI_FEW(LAI_KV_E4M3);
        default: return LAI_FEW(LAI_KV_I8);
    }
#undef LAI_FEW
}

}  // namespace
}  // namespace lai

extern "C" size_t lai_paged_attention_scratch_bytes(int head_dim) {
    if (head_dim != 64 && head_dim != 128) return 0;
    const size_t few = (size_t)lai::kMaxCtas * 2 * lai::part_floats(head_dim);
    const size_t wide = lai::paged::wide_scratch_floats(head_dim);
    return lai::kCounters * sizeof(int) + (few > wide ? few : wide) * sizeof(float);
}
extern "C" int lai_paged_attention_bf16(lai_bf16 *out, const lai_bf16 *q, int64_t ld_q,
                                        int64_t n_rows, int n_heads, const lai_paged_kv_t *kv,
                                        const lai_paged_batch_t *batch, float scale, int window,
                                        void *scratch, int *err, lai_stream_t stream) {
    return lai::attention_entry<false>(out, q, ld_q, n_rows, n_heads, kv, batch, scale, window,
                                       scratch, err, stream);
}
extern "C" int lai_paged_attention_f32(float *out, const float *q, int64_t ld_q, int64_t n_rows,
                                       int n_heads, const lai_paged_kv_t *kv,
                                       const lai_paged_batch_t *batch, float scale, int window,
                                       void *scratch, int *err, lai_stream_t stream) {
    return lai::attention_entry<true>(out, q, ld_q, n_rows, n_heads, kv, batch, scale, window,
                                      scratch, err, stream);
}
