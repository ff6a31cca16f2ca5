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
// maximum is a shuffle within the group, each global access is a whole 128- to 512-byte run, and
// both tensors' loads are in flight together. A CTA's threads cover consecutive (row, head)
// pairs; the sequence of its first row is found by counting the q_start that are not above it
// (one load per thread and a barrier, not a chain of dependent loads), and a thread walks on
// from there.
#include "paged.cuh"

namespace lai {
namespace {

using paged::Fmt;
using paged::Seq;
using paged::View;

constexpr int kThreads = 256;

template <typename T> __device__ __forceinline__ void load8(const T *p, float (&x)[8]);
template <> __device__ __forceinline__ void load8<uint16_t>(const uint16_t *p, float (&x)[8]) {
    unpack<uint16_t>(ld_stream(p), x);
}
template <> __device__ __forceinline__ void load8<float>(const float *p, float (&x)[8]) {
    float a[4], b[4];
    unpack<float>(ld_stream(p), a);
    unpack<float>(ld_stream(p + 4), b);
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
__device__ __forceinline__ uint32_t f32_to_i8(float x) {
    return (uint32_t)__float2int_rn(fminf(fmaxf(x, -127.f), 127.f)) & 0xffu;
}

// Where this thread's (row, head) lies in the cache. false: nothing to do for it (whole lane
// groups agree).
__device__ __forceinline__ bool locate(const View &a, int64_t row, int s, int head, int *err,
                                       bool first_lane, int64_t &at) {
    while (s < a.n_seqs && __ldg(a.q_start + s + 1) <= row) s++;
    if (s >= a.n_seqs) return false;
    const Seq q = paged::load_seq(a, s);
    if (row < q.row0) return false;
    const int64_t p = (int64_t)q.len - q.n + (row - q.row0);
    if (!q.ok || p < 0) {
        if (first_lane) paged::flag(err, LAI_DEVERR_POSITION);
        return false;
    }
    const int page = __ldg(a.pages + (int64_t)s * a.max_pages + (p >> a.log_page));
    if (page < 0 || page >= a.n_pages) {
        if (first_lane) paged::flag(err, LAI_DEVERR_PAGE);
        return false;
    }
    at = a.page_base(page, head) + (p & (a.page_size() - 1));
    return true;
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
    // |x| by bits: an unsigned maximum orders magnitudes and keeps an infinity or a NaN on top
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
    for (int o = HD / 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const bool finite = top < 0x7f800000u;
    float s = __fdiv_rn(__uint_as_float(top), kTop);
    s = s > 0.f ? s : 1.f;
    uint32_t w[2] = {0, 0};
    if (finite) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = __fdiv_rn(x[e], s);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float *y = x + 4 * h;
            if (FMT == LAI_KV_E4M3)
                w[h] = f32x2_to_e4m3x2(y[0], y[1]) | f32x2_to_e4m3x2(y[2], y[3]) << 16;
            else
                w[h] = f32_to_i8(y[0]) | f32_to_i8(y[1]) << 8 | f32_to_i8(y[2]) << 16 |
                       f32_to_i8(y[3]) << 24;
        }
    }
    if (!ok) return;
    *reinterpret_cast<uint2 *>(cache + at * HD + e0) = make_uint2(w[0], w[1]);
    if (e0 == 0) scale[at] = finite ? s : __int_as_float(0x7fffffff);
}

template <int HD, int FMT>
__device__ __forceinline__ void get(const unsigned char *cache, const float *scale, int64_t at,
                                    int e0, float (&x)[8]) {
    if (FMT == LAI_KV_BF16) {
        unpack<uint16_t>(ld_stream(reinterpret_cast<const uint16_t *>(cache) + at * HD + e0), x);
        return;
    }
    constexpr int kF = FMT == LAI_KV_BF16 ? LAI_KV_I8 : FMT;  // not reached for BF16
    const uint2 w = __ldg(reinterpret_cast<const uint2 *>(cache + at * HD + e0));
    const float s = __ldg(scale + at);
    const uint32_t h[4] = {paged::half2_of<kF, false>(w.x),
                           paged::half2_of<kF, true>(w.x),
                           paged::half2_of<kF, false>(w.y),
                           paged::half2_of<kF, true>(w.y)};
#pragma unroll
    for (int e = 0; e < 4; e++) {
        float lo, hi;
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
            : "=f"(lo), "=f"(hi)
            : "r"(h[e]));
        x[2 * e] = lo * s;
        x[2 * e + 1] = hi * s;
    }
}

template <typename T, int HD, int FMT>
__global__ void __launch_bounds__(kThreads)
append_kernel(const View a, const T *__restrict__ k, const T *__restrict__ v, int64_t ld, int *err) {
    constexpr int kLanes = HD / 8, kPairs = kThreads / kLanes;
    pdl_wait_prior();
    pdl_launch_dependents();
    const int64_t pair0 = (int64_t)blockIdx.x * kPairs;
    const int64_t pair = pair0 + threadIdx.x / kLanes;
    const int64_t row = pair / a.n_kv;
    const int head = (int)(pair - row * a.n_kv), e0 = (threadIdx.x % kLanes) * 8;
    float kx[8] = {}, vx[8] = {};
    if (row < a.n_rows) {  // both loads are under way while the sequence is looked up
        load8(k + row * ld + (int64_t)head * HD + e0, kx);
        load8(v + row * ld + (int64_t)head * HD + e0, vx);
    }
    const int s0 = first_seq(a, pair0 / a.n_kv);
    int64_t at = 0;
    const bool ok = row < a.n_rows && locate(a, row, s0, head, err, e0 == 0, at);
    put<HD, FMT>(a.k, a.k_scale, at, e0, kx, ok);
    put<HD, FMT>(a.v, a.v_scale, at, e0, vx, ok);
}

template <typename T, int HD, int FMT>
__global__ void __launch_bounds__(kThreads)
read_kernel(const View a, T *__restrict__ k, T *__restrict__ v, int64_t ld, int *err) {
    constexpr int kLanes = HD / 8, kPairs = kThreads / kLanes;
    pdl_wait_prior();
    pdl_launch_dependents();
    const int64_t pair0 = (int64_t)blockIdx.x * kPairs;
    const int64_t pair = pair0 + threadIdx.x / kLanes;
    const int64_t row = pair / a.n_kv;
    const int head = (int)(pair - row * a.n_kv), e0 = (threadIdx.x % kLanes) * 8;
    const int s0 = first_seq(a, pair0 / a.n_kv);
    int64_t at;
    if (row >= a.n_rows || !locate(a, row, s0, head, err, e0 == 0, at)) return;
    float kx[8], vx[8];
    get<HD, FMT>(a.k, a.k_scale, at, e0, kx);
    get<HD, FMT>(a.v, a.v_scale, at, e0, vx);
    store8(k + row * ld + (int64_t)head * HD + e0, kx);
    store8(v + row * ld + (int64_t)head * HD + e0, vx);
}

template <typename T, bool APPEND, typename P>
int rows_entry(const lai_paged_kv_t *kv, const lai_paged_batch_t *b, P k, P v, int64_t ld,
               int64_t n_rows, int *err, lai_stream_t stream) {
    View a;
    const int st = paged::check(kv, b, n_rows, &a);
    if (st != LAI_OK) return st;
    const int64_t width = (int64_t)kv->n_kv_heads * kv->head_dim;
    if (!k || !v || ld < width || ld % (16 / (int)sizeof(T)) != 0 || !aligned16(k) || !aligned16(v))
        return LAI_ERR_INVALID;
    if (n_rows == 0 || b->n_seqs == 0) return LAI_OK;
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
    const int64_t pairs = n_rows * kv->n_kv_heads, per = kThreads / (kv->head_dim / 8);
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
