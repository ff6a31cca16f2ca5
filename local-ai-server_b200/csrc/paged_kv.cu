// paged_kv.cu - writing rows of keys and values into the paged cache, and reading them back.
//
// The reference copies k and v of a token into its layer's dense F32 cache (src/tts_native.c:
// 570-574 for a prompt, :650-651 for one token). Here a row goes to page pages[s, p / page_size]
// and, for the 8-bit formats, is quantised on the way: per token and head a = max|x|,
// s = a / top (448 or 127; 1 where that is 0), c = rne(x / s) with IEEE divisions, so the stored
// bits are the ones that the definition gives and not an approximation of them.
//
// HBM bound: every row is read once and every cache row written once (and the other way round).
// A group of head_dim / 8 lanes owns one (row, head) of k and of v, 8 elements per lane, so the
// maximum is a shuffle within the group, and each global access is a whole 128- to 512-byte run.
// Measured: reading 24 sequences of 4096 E4M3 tokens, 8 heads of 128, as BF16 rows 70 us (6.0 TB/s,
// 0.93 of a copy's bandwidth); writing 40 chunks of 257 BF16 rows, 16 heads of 64, 13.8 us (4.3 TB/s:
// half of it is starting and ending). What costs time beside the bytes:
//   * The look-up of a row's place is a chain of loads (q_start, lengths, page). A CTA covers
//     consecutive (row, head) pairs, several per thread; a thread per row follows the chain and
//     leaves the place in shared memory, while an append's first rows are on their way. The
//     sequence of the CTA's first row is found by counting the q_start that are not above it (one
//     load per thread and a barrier).
//   * The divisions: 8 per lane and tensor. The scale's reciprocal is rounded correctly once, and
//     each quotient corrected twice by its remainder, q + (x - q s) (1 / s) in fused operations;
//     with a correctly rounded reciprocal and a quotient within a last place that is the correctly
//     rounded quotient (Markstein 1990). Where remainders could underflow the division itself runs.
#include "paged.cuh"

namespace lai {
namespace {

using paged::Fmt;
using paged::Seq;
using paged::View;

constexpr int kThreads = 256;

// 8 elements of a row as they are in memory.
template <typename T> struct Raw { uint4 w[sizeof(T) / 2]; };
template <typename T> __device__ __forceinline__ Raw<T> load8(const T *p) {
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) r.w[i] = ld_stream(p + i * (16 / (int)sizeof(T)));
    return r;
}
__device__ __forceinline__ void floats_of(const Raw<uint16_t> &r, float (&x)[8]) { unpack<uint16_t>(r.w[0], x); }
__device__ __forceinline__ void floats_of(const Raw<float> &r, float (&x)[8]) {
    float a[4], b[4];
    unpack<float>(r.w[0], a);
    unpack<float>(r.w[1], b);
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = a[e], x[4 + e] = b[e];
}
template <typename T> __device__ __forceinline__ void store8(T *p, const float (&x)[8]);
template <> __device__ __forceinline__ void store8<uint16_t>(uint16_t *p, const float (&x)[8]) {
    st_vec(p, pack<uint16_t>(x));
}
template <> __device__ __forceinline__ void store8<float>(float *p, const float (&x)[8]) {
    const float a[4] = {x[0], x[1], x[2], x[3]}, b[4] = {x[4], x[5], x[6], x[7]};
    st_vec(p, pack<float>(a));
    st_vec(p + 4, pack<float>(b));
}

__device__ __forceinline__ uint32_t f32x2_to_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// Four integers nearest to x (ties to even), |x| <= 127, as bytes: adding 1.5 * 2^23 leaves them in
// the low bits.
__device__ __forceinline__ uint32_t f32x4_to_i8x4(const float *x) {
    uint32_t b[4];
#pragma unroll
    for (int e = 0; e < 4; e++) b[e] = __float_as_uint(fminf(fmaxf(x[e], -127.f), 127.f) + 12582912.f);
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

// The place of a row in the cache, as the position of head 0 (a head is 1 << log_page positions),
// looking from sequence s on; -1: nowhere.
__device__ __forceinline__ int64_t place_of(const View &a, int64_t row, int s, int *err) {
    while (s < a.n_seqs && __ldg(a.q_start + s + 1) <= row) s++;
    if (s >= a.n_seqs || row >= a.n_rows) return -1;
    const Seq q = paged::load_seq(a, s);
    if (row < q.row0) return -1;
    const int p = q.len - q.n + (int)(row - q.row0);
    if (!q.ok || p < 0) {
        paged::flag(err, LAI_DEVERR_POSITION);
        return -1;
    }
    const int page = __ldg(a.pages + (int64_t)s * a.max_pages + (p >> a.log_page));
    if (page < 0 || page >= a.n_pages) {
        paged::flag(err, LAI_DEVERR_PAGE);
        return -1;
    }
    return a.page_base(page, 0) + (p & (a.page_size() - 1));
}

// The sequence that a CTA starts its search at: the number of q_start[1..] not above its row.
__device__ __forceinline__ int first_seq(const View &a, int64_t row) {
    int s = 0;
    for (int i = 0; i < a.n_seqs; i += kThreads) {
        const int j = i + threadIdx.x;
        s += __syncthreads_count(j < a.n_seqs && __ldg(a.q_start + j + 1) <= row);
    }
    return s;
}

__device__ __forceinline__ float max_abs3(float x, float y, float z) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(fabsf(x)), "f"(fabsf(y)), "f"(fabsf(z)));
    return r;
}

// Write a lane's 8 elements (and lane 0 its row's scale) where ok; all lanes take part in the
// maximum.
template <int HD, int FMT>
__device__ __forceinline__ void put(unsigned char *cache, float *scale, int64_t at, int e0,
                                    float (&x)[8], bool ok) {
    if (FMT == LAI_KV_BF16) {
        if (ok) store8(reinterpret_cast<uint16_t *>(cache) + at * HD + e0, x);
        return;
    }
    constexpr float kTop = Fmt<FMT>::kTop;
    // the largest magnitude; a NaN stays one
    float top = max_abs3(x[0], x[1], x[2]);
    top = max_abs3(top, x[3], x[4]);
    top = max_abs3(max_abs3(top, x[5], x[6]), x[7], 0.f);
#pragma unroll
    for (int o = HD / 16; o > 0; o >>= 1) top = max_abs3(top, __shfl_xor_sync(0xffffffffu, top, o), 0.f);
    const bool finite = top < __int_as_float(0x7f800000);
    float s = __fdiv_rn(top, kTop);
    s = s > 0.f ? s : 1.f;
    uint32_t w[2] = {0, 0};
    if (finite) {
        if (s > 1e-30f && s < 1e30f) {
            const float y = __frcp_rn(s);
            const float2 y2 = make_float2(y, y), ns2 = make_float2(-s, -s);
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float2 v = make_float2(x[e], x[e + 1]);
                float2 q = __fmul2_rn(v, y2);
                q = __ffma2_rn(__ffma2_rn(q, ns2, v), y2, q);
                q = __ffma2_rn(__ffma2_rn(q, ns2, v), y2, q);
                x[e] = q.x;
                x[e + 1] = q.y;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = __fdiv_rn(x[e], s);
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float *q = x + 4 * h;
            if (FMT == LAI_KV_E4M3) w[h] = f32x2_to_e4m3x2(q[0], q[1]) | f32x2_to_e4m3x2(q[2], q[3]) << 16;
            else w[h] = f32x4_to_i8x4(q);
        }
    }
    if (!ok) return;
    *reinterpret_cast<uint2 *>(cache + at * HD + e0) = make_uint2(w[0], w[1]);
    if (e0 == 0) scale[at] = finite ? s : __int_as_float(0x7fffffff);
}

// 8 stored elements and their scale, and what they stand for.
template <int FMT> struct Stored {
    uint4 w;
    float s;
};
template <int HD, int FMT>
__device__ __forceinline__ Stored<FMT> fetch(const unsigned char *cache, const float *scale, int64_t at, int e0) {
    Stored<FMT> r = {};
    if (FMT == LAI_KV_BF16) {
        r.w = ld_stream(cache + (at * HD + e0) * 2);
        return r;
    }
    const uint2 w = __ldg(reinterpret_cast<const uint2 *>(cache + at * HD + e0));
    r.w.x = w.x;
    r.w.y = w.y;
    r.s = __ldg(scale + at);
    return r;
}
template <int FMT>
__device__ __forceinline__ void values_of(const Stored<FMT> &r, float (&x)[8]) {
    if (FMT == LAI_KV_BF16) {
        unpack<uint16_t>(r.w, x);
        return;
    }
    constexpr int kF = FMT == LAI_KV_BF16 ? LAI_KV_I8 : FMT;  // not reached for BF16
    const uint32_t h[4] = {paged::half2_of<kF, false>(r.w.x), paged::half2_of<kF, true>(r.w.x),
                           paged::half2_of<kF, false>(r.w.y), paged::half2_of<kF, true>(r.w.y)};
#pragma unroll
    for (int e = 0; e < 4; e++) {
        float lo, hi;
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
            : "=f"(lo), "=f"(hi)
            : "r"(h[e]));
        x[2 * e] = lo * r.s;
        x[2 * e + 1] = hi * r.s;
    }
}

constexpr int kUnits = 4;  // (row, head) pairs per thread, kTogether of them under way at a time
constexpr int kTogether = 2;

// The pairs of a CTA: lane group i has pairs i, i + kGroups, ...
template <int HD>
struct Pairs {
    static constexpr int kLanes = HD / 8, kGroups = kThreads / kLanes, kPerCta = kGroups * kUnits;
    int64_t row0;
    int rest, n_kv;
    __device__ __forceinline__ explicit Pairs(const View &a) : n_kv(a.n_kv) {
        const int64_t pair0 = (int64_t)blockIdx.x * kPerCta;
        row0 = pair0 / n_kv;
        rest = (int)(pair0 - row0 * n_kv);
    }
    __device__ __forceinline__ int rows() const { return (rest + kPerCta - 1) / n_kv + 1; }  // touched
    // pair u of the thread: row (from row0 on) and head
    __device__ __forceinline__ int row(int u, int &head) const {
        const uint32_t i = (uint32_t)(rest + u * kGroups + (int)threadIdx.x / kLanes), r = i / (uint32_t)n_kv;
        head = (int)(i - r * n_kv);
        return (int)r;
    }
    // looks up the places of all rows; the whole CTA
    __device__ __forceinline__ void find(const View &a, int64_t *place, int *err) const {
        const int s = first_seq(a, row0);
        for (int i = threadIdx.x; i < rows(); i += kThreads) place[i] = place_of(a, row0 + i, s, err);
        __syncthreads();
    }
};

template <typename T, int HD, int FMT>
__global__ void __launch_bounds__(kThreads)
append_kernel(const View a, const T *__restrict__ k, const T *__restrict__ v, int64_t ld, int *err) {
    __shared__ int64_t place[Pairs<HD>::kPerCta + 1];
    pdl_wait_prior();
    pdl_launch_dependents();
    const Pairs<HD> pairs(a);
    const int e0 = (threadIdx.x % Pairs<HD>::kLanes) * 8;
#pragma unroll 1
    for (int u0 = 0; u0 < kUnits; u0 += kTogether) {
        Raw<T> kx[kTogether], vx[kTogether];
        int row[kTogether], head[kTogether];
#pragma unroll
        for (int u = 0; u < kTogether; u++) {
            row[u] = pairs.row(u0 + u, head[u]);
            kx[u] = vx[u] = Raw<T>{};
            if (pairs.row0 + row[u] < a.n_rows) {
                const int64_t at = (pairs.row0 + row[u]) * ld + head[u] * HD + e0;
                kx[u] = load8(k + at);
                vx[u] = load8(v + at);
            }
        }
        if (u0 == 0) pairs.find(a, place, err);
#pragma unroll
        for (int u = 0; u < kTogether; u++) {
            const int64_t p = place[row[u]], at = p + ((int64_t)head[u] << a.log_page);
            float x[8];
            floats_of(kx[u], x);
            put<HD, FMT>(a.k, a.k_scale, at, e0, x, p >= 0);
            floats_of(vx[u], x);
            put<HD, FMT>(a.v, a.v_scale, at, e0, x, p >= 0);
        }
    }
}

template <typename T, int HD, int FMT>
__global__ void __launch_bounds__(kThreads)
read_kernel(const View a, T *__restrict__ k, T *__restrict__ v, int64_t ld, int *err) {
    __shared__ int64_t place[Pairs<HD>::kPerCta + 1];
    pdl_wait_prior();
    pdl_launch_dependents();
    const Pairs<HD> pairs(a);
    const int e0 = (threadIdx.x % Pairs<HD>::kLanes) * 8;
    pairs.find(a, place, err);
#pragma unroll 1
    for (int u0 = 0; u0 < kUnits; u0 += kTogether) {
        Stored<FMT> kx[kTogether], vx[kTogether];
        int row[kTogether], head[kTogether];
#pragma unroll
        for (int u = 0; u < kTogether; u++) {
            row[u] = pairs.row(u0 + u, head[u]);
            const int64_t p = place[row[u]];
            if (p < 0) continue;
            const int64_t at = p + ((int64_t)head[u] << a.log_page);
            kx[u] = fetch<HD, FMT>(a.k, a.k_scale, at, e0);
            vx[u] = fetch<HD, FMT>(a.v, a.v_scale, at, e0);
        }
#pragma unroll
        for (int u = 0; u < kTogether; u++) {
            if (place[row[u]] < 0) continue;
            const int64_t at = (pairs.row0 + row[u]) * ld + head[u] * HD + e0;
            float x[8];
            values_of<FMT>(kx[u], x);
            store8(k + at, x);
            values_of<FMT>(vx[u], x);
            store8(v + at, x);
        }
    }
}

template <typename T, bool APPEND, typename P>
int rows_entry(const lai_paged_kv_t *kv, const lai_paged_batch_t *b, P k, P v, int64_t ld,
               int64_t n_rows, int *err, lai_stream_t stream) {
    View a;
    const int st = paged::check(kv, b, n_rows, &a);
    if (st != LAI_OK) return st;
    if (n_rows == 0 || b->n_seqs == 0) return LAI_OK;
    const int64_t width = (int64_t)kv->n_kv_heads * kv->head_dim;
    if (!k || !v || ld < width || ld % (16 / (int)sizeof(T)) != 0 || !aligned16(k) || !aligned16(v))
        return LAI_ERR_INVALID;
    const size_t nb = paged::row_bytes(n_rows, ld, width, sizeof(T));
    if (paged::hits_cache(kv, k, nb) || paged::hits_cache(kv, v, nb)) return LAI_ERR_ALIAS;
    const size_t cb = paged::cache_bytes(kv), sb = paged::scale_bytes(kv);
    // what is written must not overlap itself; k and v rows may be column blocks of one tensor
    if (APPEND && (overlaps(kv->k, cb, kv->v, cb) || (sb && overlaps(kv->k_scale, sb, kv->v_scale, sb))))
        return LAI_ERR_ALIAS;
    if (!APPEND && overlaps(k, nb, v, nb)) {
        const uintptr_t x = reinterpret_cast<uintptr_t>(k), y = reinterpret_cast<uintptr_t>(v);
        const uintptr_t d = x < y ? y - x : x - y, row = (uintptr_t)ld * sizeof(T);
        const uintptr_t w = (uintptr_t)width * sizeof(T);
        if (d % row < w || row - d % row < w) return LAI_ERR_ALIAS;
    }
    const int64_t pairs = n_rows * kv->n_kv_heads, per = kThreads / (kv->head_dim / 8) * kUnits;
    if ((pairs + per - 1) / per > INT32_MAX) return LAI_ERR_RANGE;
    const dim3 grid(grid_for(pairs, per));
    const cudaStream_t cs = as_stream(stream);
#define LAI_ROWS(HD, FMT)                                                                     \
    if constexpr (APPEND)                                                                     \
        launch_pdl(append_kernel<T, HD, FMT>, grid, dim3(kThreads), 0, cs, a, k, v, ld, err); \
    else                                                                                      \
        launch_pdl(read_kernel<T, HD, FMT>, grid, dim3(kThreads), 0, cs, a, k, v, ld, err)
#define LAI_ROWS_FMT(HD)                                                   \
    switch (kv->format) {                                                  \
        case LAI_KV_BF16: LAI_ROWS(HD, LAI_KV_BF16); break;                \
        case LAI_KV_E4M3: LAI_ROWS(HD, LAI_KV_E4M3); break;                \
        default: LAI_ROWS(HD, LAI_KV_I8); break;                           \
    }
    if (kv->head_dim == 128) {
        LAI_ROWS_FMT(128)
    } else {
        LAI_ROWS_FMT(64)
    }
#undef LAI_ROWS_FMT
#undef LAI_ROWS
    return launch_status();
}

}  // namespace
}  // namespace lai

extern "C" int lai_paged_kv_append_bf16(const lai_paged_kv_t *kv, const lai_paged_batch_t *batch,
                                        const lai_bf16 *k, const lai_bf16 *v, int64_t ld,
                                        int64_t n_rows, int *err, lai_stream_t stream) {
    return lai::rows_entry<uint16_t, true>(kv, batch, k, v, ld, n_rows, err, stream);
}
extern "C" int lai_paged_kv_append_f32(const lai_paged_kv_t *kv, const lai_paged_batch_t *batch,
                                       const float *k, const float *v, int64_t ld, int64_t n_rows,
                                       int *err, lai_stream_t stream) {
    return lai::rows_entry<float, true>(kv, batch, k, v, ld, n_rows, err, stream);
}
extern "C" int lai_paged_kv_read_bf16(lai_bf16 *k, lai_bf16 *v, int64_t ld, int64_t n_rows,
                                      const lai_paged_kv_t *kv, const lai_paged_batch_t *batch,
                                      int *err, lai_stream_t stream) {
    return lai::rows_entry<uint16_t, false>(kv, batch, k, v, ld, n_rows, err, stream);
}
extern "C" int lai_paged_kv_read_f32(float *k, float *v, int64_t ld, int64_t n_rows,
                                     const lai_paged_kv_t *kv, const lai_paged_batch_t *batch,
                                     int *err, lai_stream_t stream) {
    return lai::rows_entry<float, false>(kv, batch, k, v, ld, n_rows, err, stream);
}
