// paged.cuh - the paged key/value cache as its kernels see it: arguments, host checks, the
// ragged batch, and the 8-bit formats.
#pragma once

#include "lai_common.cuh"

namespace lai {
namespace paged {

// Formats of the cache: bytes per element, and the largest stored magnitude that a row's
// maximum is scaled to.
template <int FMT> struct Fmt;
template <> struct Fmt<LAI_KV_BF16> { static constexpr int kBytes = 2; static constexpr float kTop = 0.f; };
template <> struct Fmt<LAI_KV_E4M3> { static constexpr int kBytes = 1; static constexpr float kTop = 448.f; };
template <> struct Fmt<LAI_KV_I8> { static constexpr int kBytes = 1; static constexpr float kTop = 127.f; };

// What a kernel gets of lai_paged_kv_t and lai_paged_batch_t (both live on the host).
struct View {
    unsigned char *k, *v;
    float *k_scale, *v_scale;
    const int32_t *q_start, *kv_len, *pages;
    int64_t n_pages, n_rows;
    int log_page, n_kv, n_seqs, max_pages;

    __device__ __forceinline__ int page_size() const { return 1 << log_page; }
    // the first element of (page, head) in units of positions
    __device__ __forceinline__ int64_t page_base(int page, int head) const {
        return ((int64_t)page * n_kv + head) << log_page;
    }
};

// A sequence of the batch: its rows [row0, row0 + n) and its key count.
struct Seq {
    int row0, n, len;
    bool ok;
};
__device__ __forceinline__ Seq load_seq(const View &a, int s) {
    const int r0 = a.q_start[s], r1 = a.q_start[s + 1], len = a.kv_len[s];
    Seq q;
    q.row0 = r0;
    q.n = r1 - r0;
    q.len = len;
    q.ok = r0 >= 0 && r1 >= r0 && r1 <= a.n_rows && len >= 0 &&
           len <= ((int64_t)a.max_pages << a.log_page);
    return q;
}

__device__ __forceinline__ void flag(int *err, int bit) {
    if (err) atomicOr(err, bit);
}

// Host side: the cache and batch are well formed (what a pointer points at is checked by the
// kernels). LAI_OK, or the error the entry returns.
inline int check(const lai_paged_kv_t *kv, const lai_paged_batch_t *b, int64_t n_rows, View *out) {
    if (!kv || !b || !kv->k || !kv->v || n_rows < 0 || b->n_seqs < 0 ||
        (b->n_seqs > 0 && (!b->q_start || !b->kv_len || !b->pages)) || b->max_pages <= 0 ||
        kv->n_pages <= 0 || kv->n_kv_heads <= 0 ||
        (kv->head_dim != 64 && kv->head_dim != 128) || kv->format < LAI_KV_BF16 ||
        kv->format > LAI_KV_I8)
        return LAI_ERR_INVALID;
    const int ps = kv->page_size;
    if (ps != 16 && ps != 32 && ps != 64 && ps != 128 && ps != 256) return LAI_ERR_INVALID;
    const bool scaled = kv->format != LAI_KV_BF16;
    if (scaled != (kv->k_scale != nullptr) || scaled != (kv->v_scale != nullptr))
        return LAI_ERR_INVALID;
    if (!aligned16(kv->k) || !aligned16(kv->v) || !aligned16(kv->k_scale) || !aligned16(kv->v_scale))
        return LAI_ERR_INVALID;
    // positions and rows are 32-bit, page numbers too
    if (kv->n_pages > INT32_MAX || n_rows > INT32_MAX || kv->n_kv_heads > 65535 ||
        (int64_t)b->max_pages * ps > INT32_MAX - 1024)
        return LAI_ERR_RANGE;
    int lg = 4;
    while ((1 << lg) < ps) lg++;
    *out = View{static_cast<unsigned char *>(kv->k), static_cast<unsigned char *>(kv->v), kv->k_scale,
                kv->v_scale, b->q_start, b->kv_len, b->pages, kv->n_pages, n_rows, lg,
                kv->n_kv_heads, b->n_seqs, b->max_pages};
    return LAI_OK;
}
inline size_t cache_bytes(const lai_paged_kv_t *kv) {
    return (size_t)kv->n_pages * kv->n_kv_heads * kv->page_size * kv->head_dim *
           (kv->format == LAI_KV_BF16 ? 2 : 1);
}
inline size_t scale_bytes(const lai_paged_kv_t *kv) {
    return kv->k_scale ? (size_t)kv->n_pages * kv->n_kv_heads * kv->page_size * 4 : 0;
}
// Bytes that n_rows rows of `width` elements with stride ld reach over.
inline size_t row_bytes(int64_t n_rows, int64_t ld, int64_t width, int esize) {
    return n_rows ? ((size_t)(n_rows - 1) * ld + width) * esize : 0;
}
inline bool hits_cache(const lai_paged_kv_t *kv, const void *p, size_t n) {
    const size_t cb = cache_bytes(kv), sb = scale_bytes(kv);
    return overlaps(p, n, kv->k, cb) || overlaps(p, n, kv->v, cb) ||
           (sb && (overlaps(p, n, kv->k_scale, sb) || overlaps(p, n, kv->v_scale, sb)));
}

// ---- 8-bit values as 16-bit operands ----------------------------------------------------------
// Both formats are exact in binary16. I8: a byte b read as unsigned after flipping its top bit is
// b + 128; put under the exponent byte 0x64 it is the binary16 1024 + b + 128, and subtracting
// 1152 leaves b, exactly.
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    return __byte_perm(a, b, sel);
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// Bytes 0 and 1 (HI false) or 2 and 3 (HI true) of w as two binary16, in order.
template <int FMT, bool HI> __device__ __forceinline__ uint32_t half2_of(uint32_t w);
template <> __device__ __forceinline__ uint32_t half2_of<LAI_KV_I8, false>(uint32_t w) {
    return hsub2(prmt(w ^ 0x80808080u, 0x64646464u, 0x4140), 0x64806480u);
}
template <> __device__ __forceinline__ uint32_t half2_of<LAI_KV_I8, true>(uint32_t w) {
    return hsub2(prmt(w ^ 0x80808080u, 0x64646464u, 0x4342), 0x64806480u);
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t v) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
    return r;
}
template <> __device__ __forceinline__ uint32_t half2_of<LAI_KV_E4M3, false>(uint32_t w) {
    return e4m3x2_to_f16x2((uint16_t)(w & 0xffffu));
}
template <> __device__ __forceinline__ uint32_t half2_of<LAI_KV_E4M3, true>(uint32_t w) {
    return e4m3x2_to_f16x2((uint16_t)(w >> 16));
}

}  // namespace paged
}  // namespace lai
