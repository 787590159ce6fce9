// Attention of new tokens over a cache in pages (gsvk_op_attn_paged), for gfx950: one wave per
// (row, query head), the keys in turn, an online softmax per group of lanes.
#include <cmath>

#include "paged.h"

namespace gsvk {
namespace {

struct PagedAttn {
    PagedView kv;
    const uint16_t * q;
    int64_t q_stride;   // elements
    void * out;
    int64_t out_stride;   // elements
    float * lse;
    const int32_t * prefix;
    float scale_log2;
    int group;   // query heads per key/value head
    int window;
    int max_new;
};

// Wave of (row, head): HD / 8 lanes share a key, each holding 8 dims; the groups of lanes keep
// their own running maximum and sum and are joined at the end.
template <class T, int HD, bool F32OUT>
__global__ void __launch_bounds__(64) k_attn_paged_rows(PagedAttn a) {
    constexpr int LK = HD / 8, KI = 64 / LK;
    const int b = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 63;
    const int64_t r0 = a.kv.row0(b), r1 = a.kv.row0(b + 1);
    const int64_t row = r0 + blockIdx.x;
    if (row >= r1) return;
    const int64_t len = a.kv.keys(b);
    const int64_t p = (int64_t) a.kv.kv_len[b] - (r1 - row);
    int64_t hi = p + 1, lo = 0;
    if (a.prefix && a.prefix[b] > hi) hi = a.prefix[b];
    if (hi > len) hi = len;
    if (a.window && p - a.window + 1 > 0) lo = p - a.window + 1;

    const int sub = lane % LK, kg = lane / LK;
    float q[8];
    pg_unpack8<T>(*reinterpret_cast<const uint4 *>(a.q + row * a.q_stride + h * HD + sub * 8), q);
    float m = -INFINITY, l = 0.0f, o[8] = {};
    for (int64_t j0 = lo; j0 < hi; j0 += KI) {
        const int64_t j = j0 + kg;
        int64_t page = -1;
        if (j < hi) page = a.kv.table[b * a.kv.table_stride + (j >> a.kv.page_shift)];
        const bool see = page >= 0 && page < a.kv.n_pages;
        const int64_t at = (see ? page : 0) * a.kv.page_stride
                           + (((int64_t) (h / a.group) << a.kv.page_shift) + (j & ((1 << a.kv.page_shift) - 1))) * HD + sub * 8;
        float x[8], s = 0.0f;
        pg_unpack8<T>(*reinterpret_cast<const uint4 *>(a.kv.k + at), x);
#pragma unroll
        for (int i = 0; i < 8; i++) s = __builtin_fmaf(q[i], x[i], s);
#pragma unroll
        for (int d = 1; d < LK; d <<= 1) s += __shfl_xor(s, d, 64);
        if (!see) continue;
        s *= a.scale_log2;
        const float mn = fmaxf(m, s);
        if (mn == -INFINITY) continue;
        const float f = __builtin_amdgcn_exp2f(m - mn), e = __builtin_amdgcn_exp2f(s - mn);
        pg_unpack8<T>(*reinterpret_cast<const uint4 *>(a.kv.v + at), x);
        l = l * f + e;
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = __builtin_fmaf(e, x[i], o[i] * f);
        m = mn;
    }
    float M = m;
#pragma unroll
    for (int d = LK; d < 64; d <<= 1) M = fmaxf(M, __shfl_xor(M, d, 64));
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
    l *= f;
#pragma unroll
    for (int d = LK; d < 64; d <<= 1) l += __shfl_xor(l, d, 64);
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        o[i] *= f;
#pragma unroll
        for (int d = LK; d < 64; d <<= 1) o[i] += __shfl_xor(o[i], d, 64);
        o[i] *= inv;
    }
    if (lane >= LK) return;
    const int64_t at = row * a.out_stride + h * HD + sub * 8;
    if constexpr (F32OUT) {
        float * out = (float *) a.out + at;
        *reinterpret_cast<float4 *>(out) = make_float4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<float4 *>(out + 4) = make_float4(o[4], o[5], o[6], o[7]);
    } else {
        *reinterpret_cast<uint4 *>((uint16_t *) a.out + at) = make_uint4(pg_pack<T>(o[0], o[1]), pg_pack<T>(o[2], o[3]),
                                                                        pg_pack<T>(o[4], o[5]), pg_pack<T>(o[6], o[7]));
    }
    if (a.lse && lane == 0)
        a.lse[row * gridDim.y + h] = l != 0.0f ? 0.69314718055994531f * (M + __builtin_log2f(l)) : -INFINITY;
}

template <class T, int HD>
void launch_attn(const PagedAttn & a, int nh, bool f32, hipStream_t st) {
    const dim3 grid((unsigned) a.max_new, (unsigned) nh, (unsigned) a.kv.B);
    if (f32) hipLaunchKernelGGL((k_attn_paged_rows<T, HD, true>), grid, dim3(64), 0, st, a);
    else hipLaunchKernelGGL((k_attn_paged_rows<T, HD, false>), grid, dim3(64), 0, st, a);
}

template <class T>
void launch_attn(const PagedAttn & a, int hd, int nh, bool f32, hipStream_t st) {
    if (hd == 32) launch_attn<T, 32>(a, nh, f32, st);
    else if (hd == 64) launch_attn<T, 64>(a, nh, f32, st);
    else launch_attn<T, 128>(a, nh, f32, st);
}

}  // namespace
}  // namespace gsvk

extern "C" size_t gsvk_attn_paged_workspace_bytes(const gsvk_paged_kv * kv, int64_t tokens, int nh, int max_new,
                                                  int64_t max_keys) {
    (void) kv; (void) tokens; (void) nh; (void) max_new; (void) max_keys;
    return 0;
}

extern "C" int gsvk_op_attn_paged(const gsvk_paged_kv * kv, const void * q, int64_t tokens, int nh, int64_t q_stride,
                                  int max_new, int64_t max_keys, float scale, int window, const int32_t * prefix,
                                  void * out, int out_type, int64_t out_stride, float * lse, void * ws,
                                  size_t ws_bytes, void * stream) {
    using namespace gsvk;
    PagedAttn a{};
    GSVK_TRY(paged_view(kv, tokens, "attn_paged", a.kv));
    GSVK_REQUIRE(nh >= 1 && nh <= 65535 && nh % kv->n_kv == 0, "attn_paged: nh %d is not a multiple of n_kv %d", nh,
                 kv->n_kv);
    GSVK_REQUIRE(out_type == GSVK_TYPE_F32 || out_type == kv->type,
                 "attn_paged: out_type %d is neither F32 nor the cache's type", out_type);
    GSVK_REQUIRE(scale > 0.0f && std::isfinite(scale * 1.4426950408889634f), "attn_paged: scale must be positive and finite");
    GSVK_REQUIRE(window >= 0 && max_new >= 0 && max_keys >= 0, "attn_paged: window, max_new and max_keys must not be negative");
    if (tokens == 0 || kv->B == 0 || max_new == 0) return GSVK_OK;
    GSVK_REQUIRE(q && out, "attn_paged: q and out must be given");
    const int64_t w = (int64_t) nh * kv->hd;
    GSVK_REQUIRE((q_stride >= w && out_stride >= w) || tokens == 1, "attn_paged: a stride is smaller than its row");
    GSVK_REQUIRE((((uintptr_t) q | (uintptr_t) out) & 15) == 0 && q_stride % 8 == 0
                     && out_stride % (out_type == GSVK_TYPE_F32 ? 4 : 8) == 0,
                 "attn_paged: the rows of q and out must be 16-byte aligned");
    const size_t need = gsvk_attn_paged_workspace_bytes(kv, tokens, nh, max_new, max_keys);
    GSVK_REQUIRE(need == 0 || (ws && ws_bytes >= need && ((uintptr_t) ws & 15) == 0),
                 "attn_paged: a workspace of %zu bytes, 16-byte aligned, is needed (%zu given)", need, ws_bytes);
    a.q = (const uint16_t *) q;
    a.q_stride = q_stride;
    a.out = out;
    a.out_stride = out_stride;
    a.lse = lse;
    a.prefix = prefix;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.group = nh / kv->n_kv;
    a.window = window;
    a.max_new = max_new < tokens ? max_new : (int) tokens;
    if (kv->type == GSVK_TYPE_F16) launch_attn<PgF16>(a, kv->hd, nh, out_type == GSVK_TYPE_F32, (hipStream_t) stream);
    else launch_attn<PgBF16>(a, kv->hd, nh, out_type == GSVK_TYPE_F32, (hipStream_t) stream);
    GSVK_LAUNCH_CHECK();
    return GSVK_OK;
}
