// What the paged-cache operators share (gsvk_op_paged_append, gsvk_op_attn_paged): the cache and
// batch as the kernels see them, checked on the host, and the two 16-bit types.
#pragma once

#include "common.h"

namespace gsvk {

typedef _Float16 pg_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 pg_b8 __attribute__((ext_vector_type(8)));

// The element types of a cache. Conversions to fp32 are exact, those from it round to nearest even.
struct PgF16 {
    typedef _Float16 e;
    typedef pg_h8 v8;
    static __device__ __forceinline__ float up(uint16_t u) { return (float) __builtin_bit_cast(_Float16, u); }
};
struct PgBF16 {
    typedef __bf16 e;
    typedef pg_b8 v8;
    static __device__ __forceinline__ float up(uint16_t u) { return __uint_as_float((uint32_t) u << 16); }
};

template <class T>
__device__ __forceinline__ uint32_t pg_pack(float a, float b) {
    typedef typename T::e v2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, v2{(typename T::e) a, (typename T::e) b});
}
template <class T>
__device__ __forceinline__ void pg_unpack8(const uint4 & u, float (&x)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = T::up((uint16_t) w[i]);
        x[2 * i + 1] = T::up((uint16_t) (w[i] >> 16));
    }
}

constexpr int PG_MAX_KEYS = 1 << 26;   // of a sequence (sums of key tiles over a call stay in 31 bits)

// Batch arrays, which no store of a kernel reaches: read as constants, so that a uniform index gives
// scalar loads wherever they stand.
typedef const __attribute__((address_space(4))) int32_t pg_const;

// gsvk_paged_kv as the kernels take it. Everything that comes from device memory is checked where
// it is read: row ranges are cut to [0, tokens), page numbers to the cache.
struct PagedView {
    uint16_t * k;
    uint16_t * v;
    int64_t n_pages;
    int64_t page_stride;   // elements
    const int32_t * table;
    int64_t table_stride;
    const int32_t * seq_start;
    const int32_t * kv_len;
    int64_t tokens;
    int n_kv;
    int page_shift;
    int table_cols;
    int B;

    // the new rows of sequence b
    __device__ __forceinline__ int64_t row0(int b) const {
        const int64_t s = ((pg_const *) seq_start)[b];
        return s < 0 ? 0 : s > tokens ? tokens : s;
    }
    // keys of sequence b that the table has room for
    __device__ __forceinline__ int keys(int b) const {
        int64_t n = ((pg_const *) kv_len)[b];
        const int64_t cap = (int64_t) table_cols << page_shift;
        n = n < 0 ? 0 : n > cap ? cap : n;
        return n > PG_MAX_KEYS ? PG_MAX_KEYS : (int) n;
    }
};

// Checks the cache and batch of a call (host) and fills the view; `what` names the operator.
inline int paged_view(const gsvk_paged_kv * kv, int64_t tokens, const char * what, PagedView & o) {
    GSVK_REQUIRE(kv, "%s: kv is NULL", what);
    GSVK_REQUIRE(kv->type == GSVK_TYPE_F16 || kv->type == GSVK_TYPE_BF16, "%s: a cache is F16 or BF16 (type %d)", what,
                 kv->type);
    GSVK_REQUIRE(kv->hd == 32 || kv->hd == 64 || kv->hd == 128, "%s: head_dim %d (32, 64 and 128 are supported)", what,
                 kv->hd);
    GSVK_REQUIRE(kv->page_size >= 16 && kv->page_size <= 32768 && (kv->page_size & (kv->page_size - 1)) == 0,
                 "%s: page_size %d is not a power of two from 16 to 32768", what, kv->page_size);
    GSVK_REQUIRE(kv->n_kv >= 1 && kv->n_kv <= 65535 && kv->B >= 0 && kv->B <= 65535,
                 "%s: n_kv and B must be at most 65535 (%d, %d)", what, kv->n_kv, kv->B);
    GSVK_REQUIRE(tokens >= 0 && tokens <= INT32_MAX, "%s: tokens %lld out of range", what, (long long) tokens);
    const int64_t dense = (int64_t) kv->n_kv * kv->page_size * kv->hd;
    GSVK_REQUIRE(kv->page_stride == 0 || (kv->page_stride >= dense && kv->page_stride % 8 == 0),
                 "%s: page_stride %lld must be 0 or at least %lld and a multiple of 8", what,
                 (long long) kv->page_stride, (long long) dense);
    GSVK_REQUIRE(kv->n_pages >= 1 && kv->n_pages <= INT32_MAX, "%s: n_pages %lld out of range", what,
                 (long long) kv->n_pages);
    GSVK_REQUIRE(kv->table_cols >= 1 && kv->table_stride >= kv->table_cols && kv->table_stride <= INT32_MAX,
                 "%s: a table row has table_cols >= 1 of table_stride entries (%d, %lld)", what, kv->table_cols,
                 (long long) kv->table_stride);
    GSVK_REQUIRE(kv->B == 0 || (kv->k && kv->v && kv->table && kv->seq_start && kv->kv_len), "%s: a NULL array in kv",
                 what);
    GSVK_REQUIRE((((uintptr_t) kv->k | (uintptr_t) kv->v) & 15) == 0, "%s: k and v must be 16-byte aligned", what);
    o.k = (uint16_t *) kv->k;
    o.v = (uint16_t *) kv->v;
    o.n_pages = kv->n_pages;
    o.page_stride = kv->page_stride ? kv->page_stride : dense;
    o.table = kv->table;
    o.table_stride = kv->table_stride;
    o.seq_start = kv->seq_start;
    o.kv_len = kv->kv_len;
    o.tokens = tokens;
    o.n_kv = kv->n_kv;
    o.page_shift = __builtin_ctz((unsigned) kv->page_size);
    o.table_cols = kv->table_cols;
    o.B = kv->B;
    return GSVK_OK;
}

}  // namespace gsvk
