// paged_attention.cuh - how the paged attention kernels divide their work, and join it again.
//
// An item is a tile of up to R query rows (row = new token * group + head of the group) of one
// sequence and one kv head; its cost is the number of U-key blocks that its rows see. All items
// laid end to end are W blocks, and CTA c of N takes blocks [c W / N, (c + 1) W / N): every CTA
// reads the same number of keys however long, short or few the sequences are, and nothing has to
// be known on the host (the lengths live on the device, so a captured graph follows them). An item
// that lies in one CTA is written by it. An item cut by a CTA's border leaves (max, sum,
// accumulator) per row in the scratch, and the CTA that arrives last (a counter at the item's
// first CTA) joins the parts in their order, so the result does not depend on who was last. A CTA
// has at most two cut items: the one it starts with and the one it ends with. E blocks are added to
// every item for what starting and ending one costs, so that CTAs with many short items get fewer.
#pragma once

#include "paged.cuh"

namespace lai {
namespace paged {

constexpr int kSMs = 148;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^e for any e, held within the normal range.
__device__ __forceinline__ float pow2i(int e) {
    return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23);
}

// n / d for 0 <= n < 2^28 and d <= 16: m = ceil(2^32 / d) overshoots 2^32 / d by less than 1, so
// n m / 2^32 overshoots n / d by less than n / 2^32 < 1 / 16.
struct Div {
    uint64_t m;
    __host__ __device__ static Div by(int d) { return Div{((1ull << 32) + d - 1) / d}; }
    __device__ __forceinline__ int of(int n) const { return (int)((uint64_t)(uint32_t)n * m >> 32); }
};

struct AttnArgs {
    View kv;
    int group;      // query heads per kv head
    Div by_group;
    int window;     // 0: every earlier key
    float scale_log2;
    int64_t ld_q;
    int *counters;  // one per CTA of the grid, 0 between calls
    float *parts;   // two cut items per CTA
    int *err;
};

// An item without its kv head.
struct Tile {
    int seq, row0, q_row0;  // sequence, first flattened row in it, the sequence's first row
    int rows;               // real rows, 0: no item
    int pos0;               // position of new token 0
    int first, last;        // positions of the tile's first and last row
    int k0, k1;             // keys any row sees
    int b0, blocks;         // first block, blocks (1 for a tile that sees no key)
};

// Rows of the tile (or item) differ in which of the keys j0 .. j0 + n - 1 they see.
template <typename T>
__device__ __forceinline__ bool mixed(const T &t, int window, int j0, int n) {
    const int jf = max(j0, t.k0), jl = min(j0 + n, t.k1) - 1;
    return jl > t.first || (window && jf <= t.last - window);
}

template <int R, int U, int E>
struct Sched {
    static constexpr int kRowsPerTile = R, kBlock = U, kExtra = E;
    // Slots of tiles: sequence s has those from q_start[s] * group / R + s on, at least as many as
    // it has tiles.
    static __host__ __device__ int slots(int64_t n_rows, int group, int n_seqs) {
        return (int)(n_rows * group / R) + n_seqs;
    }
    // No batch of this shape has more blocks (they are counted in 32 bits).
    static int64_t most_blocks(const View &v, int group) {
        const int64_t keys = ((int64_t)v.max_pages << v.log_page) + U;
        return slots(v.n_rows, group, v.n_seqs) * (keys / U + 1 + E) * v.n_kv;
    }
    // (q_start never decreases here, and neither do these, wherever it leaves the rows)
    static __device__ __forceinline__ int base(const AttnArgs &a, int s) {
        return min(max(a.kv.q_start[s], 0), (int)a.kv.n_rows) * a.group / R + s;
    }
    static __device__ __forceinline__ int cost(const Tile &t) { return t.rows ? t.blocks + E : 0; }
    // The last sequence whose slots start at or before `slot` (0 if none does).
    static __device__ __forceinline__ int seq_of(const AttnArgs &a, int slot) {
        int lo = 0, hi = a.kv.n_seqs;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (base(a, mid) <= slot) lo = mid; else hi = mid;
        }
        return lo;
    }
    static __device__ __forceinline__ Tile tile(const AttnArgs &a, int slot, int s) {
        Tile t = {};
        const Seq q = load_seq(a.kv, s);
        const int i = slot - base(a, s);
        const int all = q.n * a.group;  // below 2^28 where ok
        if (!q.ok || all == 0 || i < 0 || i > (all - 1) / R) return t;
        const int r0 = i * R;
        t.seq = s;
        t.row0 = r0;
        t.q_row0 = q.row0;
        t.rows = min(R, all - r0);
        t.pos0 = q.len - q.n;
        const int first = t.pos0 + a.by_group.of(t.row0);
        const int last = t.pos0 + a.by_group.of(t.row0 + t.rows - 1);
        t.first = first;
        t.last = last;
        t.k1 = max(last + 1, 0);
        t.k0 = a.window ? max(first - a.window + 1, 0) : 0;
        t.b0 = t.k0 / U;
        t.blocks = t.k1 > t.k0 ? (t.k1 + U - 1) / U - t.b0 : 1;
        return t;
    }
};

// The sequences' rows and lengths in shared memory, where they fit: finding a CTA's work looks at
// them again and again, one load after another.
constexpr int kSeqCache = 256;
struct SeqSmem {
    int32_t q_start[kSeqCache + 1], kv_len[kSeqCache];
};
// a with its tables in shared memory (or as it is); flags sequences that are not well formed. Where
// q_start decreases there is no work at all (n_seqs 0): bisection and stepping would find different
// sequences for a slot then, and CTAs that disagree on who shares an item leave its counter behind
// for the next call. The whole CTA; has a barrier.
template <int THREADS>
__device__ __forceinline__ AttnArgs cache_seqs(const AttnArgs &a, SeqSmem &sm) {
    AttnArgs c = a;
    const bool keep = a.kv.n_seqs <= kSeqCache;
    bool falls = false;
#pragma unroll 4
    for (int s = threadIdx.x; s < a.kv.n_seqs; s += THREADS) {
        const int q0 = __ldg(a.kv.q_start + s), q1 = __ldg(a.kv.q_start + s + 1);
        falls |= q1 < q0;
        if (keep) {
            sm.q_start[s] = q0;
            sm.kv_len[s] = __ldg(a.kv.kv_len + s);
            if (s + 1 == a.kv.n_seqs) sm.q_start[s + 1] = q1;
        }
    }
    if (keep) {
        c.kv.q_start = sm.q_start;
        c.kv.kv_len = sm.kv_len;
    }
    falls = __syncthreads_or(falls);
    if (blockIdx.x == 0)
        for (int s = threadIdx.x; s < a.kv.n_seqs; s += THREADS)
            if (!load_seq(c.kv, s).ok) flag(a.err, LAI_DEVERR_POSITION);
    if (falls) c.kv.n_seqs = 0;
    return c;
}

// Where a CTA starts, and how far it goes. Positions are in blocks of the whole work.
struct Range {
    int total, ctas;  // all blocks; CTAs that have work
    int w0, w1;       // this CTA's
    int at;           // position of slot's first block
    int slot, seq, n_slots;
    // floor(total c / ctas)
    __device__ __forceinline__ int begin(int c) const {
        const int q = total / ctas, r = total - q * ctas;
        return q * c + r * c / ctas;  // r c < ctas^2
    }
    // the CTA that takes position x
    __device__ __forceinline__ int cta_of(int x) const {
        int c = (int)((float)x * ((float)ctas / (float)total));  // within 1: ctas is far below 2^22
        c = min(max(c, 0), ctas - 1);
        if (begin(c) > x) c--;
        else if (c + 1 < ctas && begin(c + 1) <= x) c++;
        return c;
    }
};

struct SchedSmem {
    int sums[32];
    int at, slot, seq;
};

template <typename S, int THREADS>
__device__ __forceinline__ Range find_range(const AttnArgs &a, SchedSmem &sm) {
    const int n_slots = S::slots(a.kv.n_rows, a.group, a.kv.n_seqs);
    const int per = (n_slots + THREADS - 1) / THREADS;
    const int s0 = min((int)threadIdx.x * per, n_slots), s1 = min(s0 + per, n_slots);
    int mine = 0, first_seq = 0;
    if (s0 < s1) {
        int s = first_seq = S::seq_of(a, s0);
#pragma unroll 1
        for (int slot = s0; slot < s1; slot++) {
            while (s + 1 < a.kv.n_seqs && S::base(a, s + 1) <= slot) s++;
            mine += S::cost(S::tile(a, slot, s));
        }
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) sm.sums[warp] = upto;
    __syncthreads();
    // every warp adds up the warps' sums
    int before = lane < THREADS / 32 ? sm.sums[lane] : 0;
    const int total = __reduce_add_sync(0xffffffffu, before);
    before = __reduce_add_sync(0xffffffffu, lane < warp ? before : 0) + upto - mine;
    Range r;
    r.total = total * a.kv.n_kv;
    r.ctas = min((int)gridDim.x, r.total);
    r.w0 = r.w1 = r.at = r.slot = r.seq = 0;
    r.n_slots = n_slots;
    if ((int)blockIdx.x >= r.ctas) return r;  // the whole CTA
    r.w0 = r.begin(blockIdx.x);
    r.w1 = r.begin(blockIdx.x + 1);
    const int nk = a.kv.n_kv;
    if (before * nk <= r.w0 && r.w0 < (before + mine) * nk) {  // one thread's slots hold w0
        int s = first_seq, at = before, slot = s0;
#pragma unroll 1
        for (; slot + 1 < s1; slot++) {
            while (s + 1 < a.kv.n_seqs && S::base(a, s + 1) <= slot) s++;
            const int c = S::cost(S::tile(a, slot, s));
            if (r.w0 < (at + c) * nk) break;
            at += c;
        }
        while (s + 1 < a.kv.n_seqs && S::base(a, s + 1) <= slot) s++;
        sm.slot = slot;
        sm.seq = s;
        sm.at = at * nk;
    }
    __syncthreads();
    r.slot = sm.slot;
    r.seq = sm.seq;
    r.at = sm.at;
    return r;
}

// The items of a CTA in order. Roles of a CTA that walk by themselves see the same ones.
template <typename S>
struct Walk {
    int at, w0, w1;          // position of the current item; the CTA's range
    int item0, item1;        // positions of the item's blocks
    Tile tl;
    int slot, seq, cost, n_slots;
    int head, blk0, blk1;    // the item's kv head; this CTA's blocks of it
    bool begins, ends;       // the item's first, last block is among them

    __device__ __forceinline__ void start(const AttnArgs &a, const Range &r) {
        w0 = r.w0;
        w1 = r.w1;
        n_slots = r.n_slots;
        slot = r.slot;
        seq = r.seq;
        tl = S::tile(a, slot, seq);
        cost = S::cost(tl);
        head = (w0 - r.at) / cost;
        at = r.at + head * cost;
    }
    // Sets the item at `at` and steps past it.
    __device__ __forceinline__ bool next(const AttnArgs &a) {
        while (at < w1) {
            if (head == a.kv.n_kv) {  // on to the next slot that holds a tile
                head = 0;
                do {
                    // the lengths must not change under the kernel; if they do, it still ends
                    if (++slot >= n_slots) return false;
                    while (seq + 1 < a.kv.n_seqs && S::base(a, seq + 1) <= slot) seq++;
                    tl = S::tile(a, slot, seq);
                    cost = S::cost(tl);
                } while (cost == 0);
            }
            item0 = at + S::kExtra;
            item1 = at + cost;
            at = item1;
            head++;
            const int lo = max(w0, item0), hi = min(item1, w1);
            if (lo >= hi) continue;  // only of the item's extra cost
            blk0 = tl.b0 + lo - item0;
            blk1 = tl.b0 + hi - item0;
            begins = lo == item0;
            ends = hi == item1;
            return true;
        }
        return false;
    }
    __device__ __forceinline__ int kv_head() const { return head - 1; }
};

// The kernel for many rows per sequence (paged_attention_wide.cu), scale_log2 > 0: LAI_OK or an
// error; and the F32 values of scratch it needs.
int attention_wide(void *out, const void *q, bool f32, int head_dim, int format, const AttnArgs &a,
                   cudaStream_t st);
size_t wide_scratch_floats(int head_dim);

}  // namespace paged
}  // namespace lai
