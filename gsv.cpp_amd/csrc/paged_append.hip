// Append of new tokens' keys and values to a cache in pages, queries and keys rotated to their
// positions on the way, for gfx950 (gsvk_op_paged_append; the dense, unrotated append it stands
// beside is part of the QKV kernels, layer.hip and qkv_attn.hip).
//
// Mathematics: a head's pair (x_i, x_j) at position p becomes (x_i c - x_j s, x_j c + x_i s) with
// c = cos[p][a], s = sin[p][a] of the pair's angle a. Everything else is copied. All in fp32, each
// result rounded once to the cache's type.
//
// Work: a unit is 16 elements of one head of one row, the 8 pairs of 8 consecutive angles, so that
// a thread reads and writes 16-byte pieces in either order of pairs: with halves the 8 elements at
// 8 u and the 8 at rot / 2 + 8 u, with neighbours the 16 at 16 u. One thread per unit, the units of
// a row (queries, keys, values in turn) consecutive. A thread finds its row's sequence by itself:
// the guess b = row (a step of one token per sequence) or a binary search in seq_start.
#include "paged.h"

namespace gsvk {
namespace {

struct AppendArgs {
    const char * q;
    const char * k;
    const char * v;
    int64_t q_stride, k_stride, v_stride;   // bytes
    uint16_t * q_out;
    const float * cos;
    const float * sin;
    const int32_t * pos;
    int64_t rope_rows;
    int32_t * n_bad;
    int nh;
    int rot;
    int pairs;
};

// the sequence of row r, or -1 for a row behind the last one
__device__ __forceinline__ int paged_seq_of(const PagedView & kv, int r) {
    if (r < kv.B && kv.seq_start[r] == r && kv.seq_start[r + 1] > r) return r;
    int lo = 0, hi = kv.B;   // the last b with seq_start[b] <= r is in [lo, hi) if there is one
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (kv.seq_start[mid] <= r) lo = mid + 1;
        else hi = mid;
    }
    return lo > 0 && r < kv.seq_start[lo] ? lo - 1 : -1;
}

// 8 elements at element offset i of a row, in fp32
template <class T, bool F32>
__device__ __forceinline__ void append_load8(const char * row, int i, float (&x)[8]) {
    if constexpr (F32) {
        const float4 a = *reinterpret_cast<const float4 *>(row + (int64_t) i * 4);
        const float4 b = *reinterpret_cast<const float4 *>(row + (int64_t) i * 4 + 16);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        pg_unpack8<T>(*reinterpret_cast<const uint4 *>(row + (int64_t) i * 2), x);
    }
}

template <class T>
__device__ __forceinline__ void append_store8(uint16_t * p, const float (&x)[8]) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pg_pack<T>(x[0], x[1]), pg_pack<T>(x[2], x[3]),
                                               pg_pack<T>(x[4], x[5]), pg_pack<T>(x[6], x[7]));
}

constexpr int AP_THREADS = 256;

template <class T, bool F32, int HD>
__global__ void __launch_bounds__(AP_THREADS) k_paged_append(PagedView kv, AppendArgs a) {
    constexpr int UH = HD / 16;   // units per head
    const int per_row = (a.nh + 2 * kv.n_kv) * UH;
    const int64_t id = (int64_t) blockIdx.x * AP_THREADS + threadIdx.x;
    const int64_t row = id / per_row;
    if (row >= kv.tokens) return;
    const int unit = (int) (id - row * per_row), head = unit / UH, u = unit % UH;

    const int b = paged_seq_of(kv, (int) row);
    if (b < 0) return;
    // n rows end at key kv_len - 1
    const int64_t slot = (int64_t) kv.kv_len[b] - (kv.seq_start[b + 1] - row);
    const int64_t p = a.pos ? a.pos[row] : slot;
    const int64_t col = slot >> kv.page_shift;
    int64_t page = -1;
    if (slot >= 0 && slot < PG_MAX_KEYS && col < kv.table_cols) page = kv.table[b * kv.table_stride + col];
    if (page < 0 || page >= kv.n_pages || (a.cos && (p < 0 || p >= a.rope_rows))) {
        if (unit == 0 && a.n_bad) atomicAdd(a.n_bad, 1);
        return;
    }
    const int kh = head - a.nh, vh = kh - kv.n_kv;   // the key or value head
    const char * src = kh < 0 ? a.q + row * a.q_stride : vh < 0 ? a.k + row * a.k_stride : a.v + row * a.v_stride;
    const int from = (kh < 0 ? head : vh < 0 ? kh : vh) * HD;
    uint16_t * dst;
    if (kh < 0) {
        dst = a.q_out + (row * a.nh + head) * HD;
    } else {
        const int64_t at = page * kv.page_stride + (((int64_t) (vh < 0 ? kh : vh) << kv.page_shift)
                                                    + (slot & ((1 << kv.page_shift) - 1))) * HD;
        dst = (vh < 0 ? kv.k : kv.v) + at;
    }
    const bool turn = vh < 0 && 16 * u < a.rot;
    // the unit's two pieces of 8: x and y are the pairs' first and second elements with halves,
    // the first and last four pairs with neighbours
    const int i0 = turn && !a.pairs ? 8 * u : 16 * u;
    const int i1 = turn && !a.pairs ? (a.rot >> 1) + 8 * u : 16 * u + 8;
    float x[8], y[8];
    append_load8<T, F32>(src, from + i0, x);
    append_load8<T, F32>(src, from + i1, y);
    if (turn) {
        const int64_t at = p * (a.rot >> 1) + 8 * u;
        float c[8], s[8];
        append_load8<T, true>(reinterpret_cast<const char *>(a.cos + at), 0, c);
        append_load8<T, true>(reinterpret_cast<const char *>(a.sin + at), 0, s);
        if (!a.pairs) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float f = x[i], g = y[i];
                x[i] = __builtin_fmaf(f, c[i], -(g * s[i]));
                y[i] = __builtin_fmaf(g, c[i], f * s[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float f = x[2 * i], g = x[2 * i + 1];
                x[2 * i] = __builtin_fmaf(f, c[i], -(g * s[i]));
                x[2 * i + 1] = __builtin_fmaf(g, c[i], f * s[i]);
                const float d = y[2 * i], e = y[2 * i + 1];
                y[2 * i] = __builtin_fmaf(d, c[4 + i], -(e * s[4 + i]));
                y[2 * i + 1] = __builtin_fmaf(e, c[4 + i], d * s[4 + i]);
            }
        }
    }
    append_store8<T>(dst + i0, x);
    append_store8<T>(dst + i1, y);
}

template <class T, bool F32>
void launch_append(const PagedView & kv, const AppendArgs & a, int hd, hipStream_t st) {
    const int64_t units = kv.tokens * (a.nh + 2 * kv.n_kv) * (hd / 16);
    const dim3 grid((unsigned) ((units + AP_THREADS - 1) / AP_THREADS));
    if (hd == 32) hipLaunchKernelGGL((k_paged_append<T, F32, 32>), grid, dim3(AP_THREADS), 0, st, kv, a);
    else if (hd == 64) hipLaunchKernelGGL((k_paged_append<T, F32, 64>), grid, dim3(AP_THREADS), 0, st, kv, a);
    else hipLaunchKernelGGL((k_paged_append<T, F32, 128>), grid, dim3(AP_THREADS), 0, st, kv, a);
}

}  // namespace
}  // namespace gsvk

extern "C" int gsvk_op_paged_append(const gsvk_paged_kv * kv, const void * q, const void * k, const void * v,
                                    int x_type, int64_t tokens, int nh, int64_t q_stride, int64_t k_stride,
                                    int64_t v_stride, const gsvk_rope * rope, void * q_out, int32_t * n_bad,
                                    void * stream) {
    using namespace gsvk;
    PagedView view;
    GSVK_TRY(paged_view(kv, tokens, "paged_append", view));
    GSVK_REQUIRE(x_type == GSVK_TYPE_F32 || x_type == kv->type,
                 "paged_append: x_type %d is neither F32 nor the cache's type", x_type);
    GSVK_REQUIRE(nh >= 0 && nh <= 65535, "paged_append: nh %d out of range", nh);
    if (tokens == 0 || kv->B == 0) return GSVK_OK;   // (an empty array may be NULL)
    GSVK_REQUIRE((nh > 0) == (q != nullptr) && (q != nullptr) == (q_out != nullptr),
                 "paged_append: q, q_out and nh go together");
    GSVK_REQUIRE(k && v, "paged_append: k and v must be given");
    const int64_t es = x_type == GSVK_TYPE_F32 ? 4 : 2;
    GSVK_REQUIRE((!q || q_stride >= (int64_t) nh * kv->hd || tokens == 1)
                     && ((k_stride >= (int64_t) kv->n_kv * kv->hd && v_stride >= (int64_t) kv->n_kv * kv->hd) || tokens == 1),
                 "paged_append: a stride is smaller than its row");
    GSVK_REQUIRE((((uintptr_t) q | (uintptr_t) k | (uintptr_t) v | (uintptr_t) q_out) & 15) == 0
                     && (((q ? q_stride : 0) | k_stride | v_stride) * es) % 16 == 0,
                 "paged_append: rows must be 16-byte aligned");
    GSVK_REQUIRE(q_out != q || !q || (x_type == kv->type && q_stride == (int64_t) nh * kv->hd),
                 "paged_append: q_out may be q only where q is dense and of the cache's type");
    AppendArgs a{};
    if (rope) {
        GSVK_REQUIRE(rope->cos && rope->sin && rope->rows >= 1, "paged_append: rope without tables");
        GSVK_REQUIRE(rope->rot >= 16 && rope->rot % 16 == 0 && rope->rot <= kv->hd,
                     "paged_append: rot %d is not a multiple of 16 up to head_dim %d", rope->rot, kv->hd);
        GSVK_REQUIRE((((uintptr_t) rope->cos | (uintptr_t) rope->sin) & 15) == 0,
                     "paged_append: cos and sin must be 16-byte aligned");
        a.cos = rope->cos;
        a.sin = rope->sin;
        a.pos = rope->pos;
        a.rope_rows = rope->rows;
        a.rot = rope->rot;
        a.pairs = rope->pairs != 0;
    }
    GSVK_REQUIRE(tokens * (nh + 2 * (int64_t) kv->n_kv) * (kv->hd / 16) <= (int64_t) UINT32_MAX - AP_THREADS,
                 "paged_append: too many elements for one launch");
    a.q = (const char *) q;
    a.k = (const char *) k;
    a.v = (const char *) v;
    a.q_stride = q_stride * es;
    a.k_stride = k_stride * es;
    a.v_stride = v_stride * es;
    a.q_out = (uint16_t *) q_out;
    a.n_bad = n_bad;
    a.nh = nh;
    hipStream_t st = (hipStream_t) stream;
    if (kv->type == GSVK_TYPE_F16) {
        if (x_type == GSVK_TYPE_F32) launch_append<PgF16, true>(view, a, kv->hd, st);
        else launch_append<PgF16, false>(view, a, kv->hd, st);
    } else {
        if (x_type == GSVK_TYPE_F32) launch_append<PgBF16, true>(view, a, kv->hd, st);
        else launch_append<PgBF16, false>(view, a, kv->hd, st);
    }
    GSVK_LAUNCH_CHECK();
    return GSVK_OK;
}
