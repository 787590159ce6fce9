// Attention of new tokens over a cache in pages (gsvk_op_attn_paged), for gfx950.
//
// Rows. The query heads that share a key/value head are rows of one product: of the n new tokens
// of a sequence, row r = token r / G, head r % G of the group of G. A row at key index p sees
// [max(0, p - window + 1), min(keys, max(p + 1, prefix))); both ends grow with the token, so a
// tile's first and last row give its ranges.
//
// Both kernels form the scores transposed, S^T[key][row] = K . Q^T, so that a lane holds one row
// and several keys: the softmax of a row is in-lane work plus an exchange with the lanes that hold
// its other keys, and the registers of P^T are the operand of O^T[dim][row] += V^T . P^T as they
// are (the keys of a step in the order of the score registers; V^T is read from LDS in that order
// by the transposing 16-bit read, four keys of one dim per lane).
//
//   k_attn_paged_few    sequences of at most 32 rows (single tokens, drafts): the keys are dealt to
//                       the 4 or 8 waves of a workgroup in blocks of 32, each wave with its own running
//                       maximum and sum; K goes straight into the operand registers
//                       (v_mfma_f32_16x16x32: 16 keys x 32 dims), V through a tile of LDS that
//                       belongs to the wave, so the loop has no barrier. Bound by HBM.
//   k_attn_paged_chunk  longer chunks: 4 waves of 32 rows share key tiles of 64 in LDS (double
//                       buffered), v_mfma_f32_32x32x16.
// Where that makes too few workgroups keys are divided too: k_attn_paged_few cuts each row tile into
// nsplit runs of keys, k_attn_paged_balanced all row tiles together into equal runs; (maximum, sum,
// unnormalised output) of the parts are joined by k_attn_paged_join. Where there are enough, but unequal
// ones, k_attn_paged_balanced starts them from the longest to the shortest.
//
// Softmax. Exponents are base 2. The reference exponent m of a row is not its running maximum but
// follows it: it is moved (and O, l rescaled) only when a score exceeds it by more than 2^12, to
// 2^4 above. Sums and outputs are relative to m throughout, so the result is that of any m;
// probabilities stay below 2^12, in range of fp16, and those far below the maximum are kept from
// its subnormals. They are rounded to the cache's type for the product (half a step each, random
// in sign: on the output about as much again as its own rounding); l sums them unrounded.
//
// What a row does not see must not reach it. Scores of unseen keys are replaced by -inf. Values
// of keys that no row of the tile sees are replaced by zeros on their way to LDS. Where some rows
// of a tile see a key and others do not, 0 * inf would still give NaN: such blocks are searched
// for infinities and NaNs, which are taken out of the product and added to the rows that see them
// (rare; a positive probability times an infinity is that infinity).
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "paged.h"

namespace gsvk {
namespace {

typedef float pg_f4 __attribute__((ext_vector_type(4)));
typedef float pg_f16 __attribute__((ext_vector_type(16)));
typedef short pg_s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) pg_s4 pg_lds4;
typedef __attribute__((address_space(3))) uint16_t pg_lds1;

constexpr int FEW_ROWS = 32;          // rows of a sequence up to which k_attn_paged_few takes it
constexpr int FEW_KEYS = 32;
constexpr int CH_WAVES = 4, CH_KEYS = 64, CH_ROWS = CH_WAVES * 32;
constexpr float M_NONE = -FLT_MAX;    // m of a row that has seen nothing: exp2(score - m) of -inf is 0
constexpr float M_ROOM = 12.0f, M_SET = 4.0f;

struct BalHead;
struct BalTile;

struct PagedAttn {
    PagedView kv;
    const uint16_t * q;
    int64_t q_stride;   // elements
    void * out;
    int64_t out_stride;   // elements
    float * lse;
    const int32_t * prefix;
    float * part_o;     // [nsplit][tokens * nh][HD]
    float * part_ml;    // [nsplit][tokens * nh][2]
    BalHead * bal_head;   // k_attn_paged_balanced's tables and slots
    BalTile * bal_tiles;
    float * bal_part;
    float scale_log2;
    int group;   // query heads per key/value head
    int window;
    int max_new;
    int out_f32;
    int nsplit;         // runs that a sequence of few rows is cut into
    int min_rows;       // of a chunk: sequences of fewer rows are few_tile's
    int chunk_groups;   // workgroups of chunks
    int bal_most;       // row tiles of a head that there can be (k_attn_paged_balanced)
    int ordered;        // k_attn_paged_balanced: whole row tiles by length
    int few_rows;       // rows that a sequence of few rows can have
};

template <class T>
__device__ __forceinline__ pg_f4 mfma16(typename T::v8 a, typename T::v8 b, pg_f4 c) {
    if constexpr (__is_same(T, PgF16)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
template <class T>
__device__ __forceinline__ pg_f16 mfma32(typename T::v8 a, typename T::v8 b, pg_f16 c) {
    if constexpr (__is_same(T, PgF16)) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Transposing LDS read: the 16 lanes of a group give the addresses of 4 rows x 16 columns of
// 16-bit values (lane i: row i / 4, columns 4 (i % 4) .. + 3), lane i receives column i of the 4 rows.
__device__ __forceinline__ uint2 lds_tr4(const uint16_t * p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((pg_lds4 *) p));
}
template <class T>
__device__ __forceinline__ typename T::v8 v8_of(uint2 a, uint2 b) {
    return __builtin_bit_cast(typename T::v8, make_uint4(a.x, a.y, b.x, b.y));
}
template <class T>
__device__ __forceinline__ typename T::v8 v8_of(const uint4 & a) { return __builtin_bit_cast(typename T::v8, a); }

// max / sum with the lane 32 away
__device__ __forceinline__ float max_x32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_x32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Swizzles of 16-byte pieces inside a key's LDS row of HD values, so that what 32 lanes read falls in
// different banks (256 bytes): for K 16 bytes of 16 keys, for V (read transposed) 32 bytes of 8 keys
// with the 16-row products, 64 bytes of 4 keys with the 32-row ones.
template <int HD>
__device__ __forceinline__ int swz_v(int key) { return 2 * ((key / (128 / HD)) & (HD / 16 - 1)); }
template <int HD>
__device__ __forceinline__ int swz_vc(int key) { return 4 * ((key / (128 / HD)) & (HD / 32 - 1)); }
template <int HD>
__device__ __forceinline__ int swz_k(int key) { return (key / (128 / HD)) & (HD / 8 - 1); }

// infinities and NaNs of a pair of 16-bit values: all exponent bits set
template <class T>
__device__ __forceinline__ uint32_t odd_mask(uint32_t w) {
    constexpr uint32_t E = __is_same(T, PgF16) ? 0x7C007C00u : 0x7F807F80u, ONE = E & ~(E << 1);
    return ((w & E) + ONE) & 0x80008000u;   // (no carry leaves a half: its sign bit was cleared)
}
template <class T>
__device__ __forceinline__ bool any_odd(const uint4 & u) {
    return (odd_mask<T>(u.x) | odd_mask<T>(u.y) | odd_mask<T>(u.z) | odd_mask<T>(u.w)) != 0;
}
template <class T>
__device__ __forceinline__ void clear_odd(uint4 & u) {
    uint32_t * w = &u.x;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t o = odd_mask<T>(w[i]);
        w[i] &= ~((o >> 15) * 0xffffu);
    }
}
template <class T>
__device__ __forceinline__ bool is_odd(uint16_t u) { return odd_mask<T>(u) != 0; }

// What a workgroup works on: its sequence's rows and the key ranges of rows
struct Seq {
    int64_t row0;   // first row of the token arrays
    int n;          // new tokens that are computed
    int rows;       // n * G
    int keys;
    int64_t p0;     // key index of token 0 (may be negative)
    int prefix;
};

__device__ __forceinline__ Seq seq_of(const PagedAttn & a, int b) {
    Seq s;
    s.row0 = a.kv.row0(b);
    const int64_t n = a.kv.row0(b + 1) - s.row0;
    s.keys = a.kv.keys(b);
    s.p0 = (int64_t) ((pg_const *) a.kv.kv_len)[b] - n;
    s.n = n < 0 ? 0 : n > a.max_new ? a.max_new : (int) n;
    s.rows = s.n * a.group;
    s.prefix = a.prefix ? ((pg_const *) a.prefix)[b] : 0;
    return s;
}
__device__ __forceinline__ int key_lo(const PagedAttn & a, const Seq & s, int tok) {
    const int64_t lo = s.p0 + tok - a.window + 1;
    return a.window && lo > 0 ? (int) lo : 0;
}
__device__ __forceinline__ int key_hi(const Seq & s, int tok) {
    int64_t hi = s.p0 + tok + 1;
    hi = hi > s.prefix ? hi : s.prefix;
    return hi < 0 ? 0 : hi > s.keys ? s.keys : (int) hi;
}

// Page of a key (uniform over the wave), -1 if it has none
__device__ __forceinline__ int page_of(const PagedAttn & a, pg_const * tb, int key) {
    const int col = key >> a.kv.page_shift;
    const int pg = col < a.kv.table_cols ? tb[col] : -1;
    return pg >= 0 && pg < a.kv.n_pages ? pg : -1;
}
// Element offset of key `key` (on page pg; any page if it has none) of head kvh
template <int HD>
__device__ __forceinline__ int64_t key_at(const PagedAttn & a, int pg, int kvh, int key) {
    return (int64_t) max(pg, 0) * a.kv.page_stride
           + (((int64_t) kvh << a.kv.page_shift) + (key & ((1 << a.kv.page_shift) - 1))) * HD;
}

// Store 8 output values of a row
template <class T>
__device__ __forceinline__ void store8(const PagedAttn & a, int64_t row, int col, const float (&x)[8]) {
    const int64_t at = row * a.out_stride + col;
    if (a.out_f32) {
        float4 * o = reinterpret_cast<float4 *>((float *) a.out + at);
        o[0] = make_float4(x[0], x[1], x[2], x[3]);
        o[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        *reinterpret_cast<uint4 *>((uint16_t *) a.out + at) = make_uint4(pg_pack<T>(x[0], x[1]), pg_pack<T>(x[2], x[3]),
                                                                        pg_pack<T>(x[4], x[5]), pg_pack<T>(x[6], x[7]));
    }
}
template <class T>
__device__ __forceinline__ void store4(const PagedAttn & a, int64_t row, int col, float x, float y, float z, float w) {
    const int64_t at = row * a.out_stride + col;
    if (a.out_f32) *reinterpret_cast<float4 *>((float *) a.out + at) = make_float4(x, y, z, w);
    else *reinterpret_cast<uint2 *>((uint16_t *) a.out + at) = make_uint2(pg_pack<T>(x, y), pg_pack<T>(z, w));
}
// natural logarithm of a row's sum (l relative to 2^m)
__device__ __forceinline__ float lse_of(float m, float l) {
    return l != 0.0f ? 0.69314718055994531f * (m + __builtin_log2f(l)) : -INFINITY;
}

// ---- few rows ------------------------------------------------------------------------------------

// LDS of a wave (V tile, then outputs) and of a workgroup
template <int HD>
constexpr int few_wave_lds() { return FEW_KEYS * HD * 2 > 16 * (HD + 4) * 4 ? FEW_KEYS * HD * 2 : 16 * (HD + 4) * 4; }
template <int HD, int QT, int NW>
struct FewLds {
    char mem[NW * few_wave_lds<HD>()];
    float ml[NW][QT * 16][2];
};

// QT tiles of 16 rows (row tile rt) of (head kvh, sequence b), keys of one of nsplit runs, by a workgroup
// of NW waves; sequences of more than FEW_ROWS rows are chunks
template <class T, int HD, int QT, int NW>
__device__ __forceinline__ void few_tile(const PagedAttn & a, int b, int kvh, int rt, int split,
                                         FewLds<HD, QT, NW> & lds) {
    constexpr int C = HD / 8, NV = FEW_KEYS * C / 64, NK = HD / 32, DT = HD / 16, OS = HD + 4;
    constexpr int VB = few_wave_lds<HD>();
    char * s_mem = lds.mem;
    auto & s_ml = lds.ml;

    const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Seq s = seq_of(a, b);
    const int r0 = rt * QT * 16;
    if (r0 >= s.rows || s.rows > FEW_ROWS) return;
    const int nh = a.group * a.kv.n_kv;
    const int tok0 = r0 / a.group, tok1 = min(r0 + QT * 16, s.rows) - 1, tokl = tok1 / a.group;
    const int klo = key_lo(a, s, tok0), khi = key_hi(s, tokl);
    const int lo_max = key_lo(a, s, tokl), hi_min = key_hi(s, tok0);

    int lo[QT], hi[QT];
    typename T::v8 qf[QT][NK];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const int r = min(r0 + t * 16 + li, s.rows - 1), tok = r / a.group, h = kvh * a.group + r % a.group;
        lo[t] = key_lo(a, s, tok);
        hi[t] = key_hi(s, tok);
        const uint16_t * qp = a.q + (s.row0 + tok) * a.q_stride + h * HD + 8 * lg;
#pragma unroll
        for (int c = 0; c < NK; c++) qf[t][c] = v8_of<T>(*reinterpret_cast<const uint4 *>(qp + 32 * c));
    }

    // the run of key blocks of this split, dealt to the waves in turn
    const int blk_a = klo / FEW_KEYS, nblk = khi > klo ? (khi + FEW_KEYS - 1) / FEW_KEYS - blk_a : 0;
    const int per = (nblk + a.nsplit - 1) / a.nsplit;
    const int blk0 = blk_a + min(nblk, split * per), blk1 = blk_a + min(nblk, (split + 1) * per);

    pg_const * tb = (pg_const *) (a.kv.table + b * a.kv.table_stride);
    uint16_t * sv = reinterpret_cast<uint16_t *>(s_mem + wave * VB);
    uint4 kr[2][NK], vr[NV];
    int pg[2];
    const auto fetch = [&](int blk, const int (&p)[2]) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int64_t at = key_at<HD>(a, p[t], kvh, blk * FEW_KEYS + 16 * t);
            const uint16_t * kp = a.kv.k + at + li * HD + 8 * lg;
            const uint16_t * vp = a.kv.v + at + lane * 8;
#pragma unroll
            for (int c = 0; c < NK; c++) kr[t][c] = *reinterpret_cast<const uint4 *>(kp + 32 * c);
#pragma unroll
            for (int i = 0; i < NV / 2; i++) vr[t * (NV / 2) + i] = *reinterpret_cast<const uint4 *>(vp + i * 512);
        }
    };

    float m[QT], l[QT];
    pg_f4 o[QT][DT];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        m[t] = M_NONE;
        l[t] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++) o[t][d] = pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    int blk = blk0 + wave;
    if (blk < blk1) {
        pg[0] = page_of(a, tb, blk * FEW_KEYS);
        pg[1] = page_of(a, tb, blk * FEW_KEYS + 16);
        fetch(blk, pg);
    }
    for (; blk < blk1; blk += NW) {
        const int kb = blk * FEW_KEYS;
        const bool ok0 = pg[0] >= 0, ok1 = pg[1] >= 0;
        const bool full = kb >= lo_max && kb + FEW_KEYS <= hi_min && ok0 && ok1;
        // the next block's pages
        const int nb = blk + NW < blk1 ? blk + NW : blk;
        const int np[2] = {page_of(a, tb, nb * FEW_KEYS), page_of(a, tb, nb * FEW_KEYS + 16)};
        bool odd = false;
        if (!full) {
            const bool ragged = lo_max > klo || hi_min < khi;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int key = kb + (i * 64 + lane) / C;
                const bool see = key >= klo && key < khi && (i < NV / 2 ? ok0 : ok1);
                if (!see) vr[i] = make_uint4(0, 0, 0, 0);
                if (ragged) odd |= any_odd<T>(vr[i]);
            }
            odd = __any(odd);
            if (odd)
#pragma unroll
                for (int i = 0; i < NV; i++) clear_odd<T>(vr[i]);
        }
        // scores
        pg_f4 sc[QT][2];
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int t = 0; t < QT; t++) {
                sc[t][k] = pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < NK; c++) sc[t][k] = mfma16<T>(v8_of<T>(kr[k][c]), qf[t][c], sc[t][k]);
            }
        // V into the wave's LDS tile, the next block on its way
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int u = i * 64 + lane, key = u / C;
            *reinterpret_cast<uint4 *>(sv + key * HD + (((u % C) ^ swz_v<HD>(key)) << 3)) = vr[i];
        }
        pg[0] = np[0];
        pg[1] = np[1];
        fetch(nb, pg);
        typename T::v8 pf[QT];
#pragma unroll
        for (int t = 0; t < QT; t++) {
            if (!full) {
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const int key = kb + 16 * k + 4 * lg + v;
                        if (!(key >= lo[t] && key < hi[t] && (k ? ok1 : ok0))) sc[t][k][v] = -INFINITY;
                    }
            }
            float top = fmaxf(fmaxf(fmaxf(sc[t][0][0], sc[t][0][1]), fmaxf(sc[t][0][2], sc[t][0][3])),
                              fmaxf(fmaxf(sc[t][1][0], sc[t][1][1]), fmaxf(sc[t][1][2], sc[t][1][3])));
            top *= a.scale_log2;
            if (__any(top > m[t] + M_ROOM)) {
                top = max_x32(fmaxf(top, __shfl_xor(top, 16, 64)));
                const float mn = fmaxf(m[t], top - M_SET);
                const float f = __builtin_amdgcn_exp2f(m[t] - mn);
                m[t] = mn;
                l[t] *= f;
#pragma unroll
                for (int d = 0; d < DT; d++) o[t][d] *= f;
            }
            float p[8], sum = 0.0f;
#pragma unroll
            for (int v = 0; v < 8; v++) {
                p[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][v >> 2][v & 3], a.scale_log2, -m[t]));
                sum += p[v];
            }
            l[t] += sum;
            pf[t] = v8_of<T>(make_uint4(pg_pack<T>(p[0], p[1]), pg_pack<T>(p[2], p[3]), pg_pack<T>(p[4], p[5]),
                                        pg_pack<T>(p[6], p[7])));
        }
        // O^T += V^T . P^T, keys 4 g + .. of both halves
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const int key = 4 * lg + (li >> 2), ch = 2 * d + ((li & 3) >> 1);
            const uint16_t * p = sv + key * HD + ((ch ^ swz_v<HD>(key)) << 3) + 4 * (li & 1);
            const uint16_t * p2 = sv + (key + 16) * HD + ((ch ^ swz_v<HD>(key + 16)) << 3) + 4 * (li & 1);
            const typename T::v8 vf = v8_of<T>(lds_tr4(p), lds_tr4(p2));
#pragma unroll
            for (int t = 0; t < QT; t++) o[t][d] = mfma16<T>(vf, pf[t], o[t][d]);
        }
        if (odd) {   // the infinities and NaNs that some of the rows see
            for (int j = 0; j < FEW_KEYS; j++) {
                const int key = kb + j, page = page_of(a, tb, key);
                if (page < 0 || key < klo || key >= khi) continue;
                const uint16_t * vp = a.kv.v + key_at<HD>(a, page, kvh, key) + 4 * lg;
#pragma unroll
                for (int t = 0; t < QT; t++) {
                    const bool see = key >= lo[t] && key < hi[t];
#pragma unroll
                    for (int d = 0; d < DT; d++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint16_t u = vp[16 * d + e];
                            if (see && is_odd<T>(u)) o[t][d][e] += T::up(u);
                        }
                }
            }
        }
    }

    // join the waves
#pragma unroll
    for (int t = 0; t < QT; t++) {
        l[t] = sum_x32(l[t] + __shfl_xor(l[t], 16, 64));
        if (lg == 0) {
            s_ml[wave][t * 16 + li][0] = m[t];
            s_ml[wave][t * 16 + li][1] = l[t];
        }
    }
    __syncthreads();
    float * so = reinterpret_cast<float *>(s_mem);
    for (int t = 0; t < QT; t++) {
        if (t) __syncthreads();
        float M = s_ml[0][t * 16 + li][0];
#pragma unroll
        for (int w = 1; w < NW; w++) M = fmaxf(M, s_ml[w][t * 16 + li][0]);
        const float f = __builtin_amdgcn_exp2f(s_ml[wave][t * 16 + li][0] - M);
#pragma unroll
        for (int d = 0; d < DT; d++) {
            pg_f4 x = QT == 1 || t == 0 ? o[0][d] : o[QT - 1][d];
            x *= f;
            *reinterpret_cast<pg_f4 *>(so + (wave * 16 + li) * OS + 16 * d + 4 * lg) = x;
        }
        __syncthreads();
        // a thread: 8 dims of a row
        const int rr = tid / C, col = (tid % C) * 8, r = r0 + t * 16 + rr;
        if (rr < 16 && r < s.rows) {
            const int tok = r / a.group, h = kvh * a.group + r % a.group;
            float Mr = M_NONE, L = 0.0f, x[8] = {};
#pragma unroll
            for (int w = 0; w < NW; w++) Mr = fmaxf(Mr, s_ml[w][t * 16 + rr][0]);
#pragma unroll
            for (int w = 0; w < NW; w++) {
                L += s_ml[w][t * 16 + rr][1] * __builtin_amdgcn_exp2f(s_ml[w][t * 16 + rr][0] - Mr);
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] += so[(w * 16 + rr) * OS + col + i];
            }
            const int64_t row = s.row0 + tok, id = row * nh + h;
            if (a.nsplit == 1) {
                const float inv = L != 0.0f ? 1.0f / L : 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = L != 0.0f ? x[i] * inv : 0.0f;
                store8<T>(a, row, h * HD + col, x);
                if (a.lse && col == 0) a.lse[id] = lse_of(Mr, L);
            } else {
                const int64_t at = (int64_t) split * a.kv.tokens * nh + id;
                float4 * po = reinterpret_cast<float4 *>(a.part_o + at * HD + col);
                po[0] = make_float4(x[0], x[1], x[2], x[3]);
                po[1] = make_float4(x[4], x[5], x[6], x[7]);
                if (col == 0) *reinterpret_cast<float2 *>(a.part_ml + 2 * at) = make_float2(Mr, L);
            }
        }
    }
}

// Calls whose sequences all have few rows
template <class T, int HD, int QT, int NW>
__global__ void __launch_bounds__(NW * 64, 2) k_attn_paged_few(PagedAttn a) {
    __shared__ __align__(16) FewLds<HD, QT, NW> lds;
    few_tile<T, HD, QT, NW>(a, blockIdx.z, blockIdx.y, blockIdx.x / a.nsplit, blockIdx.x % a.nsplit, lds);
}

// ---- chunks ----------------------------------------------------------------------------------------

// A wave's direct load of 1 KB: lane L's 16 bytes at base + off (bytes) to lds + 16 L. In asm, since the
// compiler waits for every direct load in flight before any LDS read that it cannot tell apart
// from their targets (and the tile after this one is in flight while this one is read). No outputs;
// the waits are wait_loads'. The s_nop is the wait state between a write of m0 and a load that reads it.
__device__ __forceinline__ void load_lds(const char * base, uint32_t off, uint16_t * lds) {
#ifdef GSVK_HOSTEMU
    __builtin_amdgcn_global_load_lds(base + off, (pg_lds1 *) lds, 16, 0, 0);
#else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"((uint32_t) (uintptr_t) (pg_lds1 *) lds), "v"(off), "s"(base)
                 : "memory");
#endif
}
// Every load of this wave has landed, every LDS operation of it is done (gfx9 encoding: vmcnt in bits
// 3:0 and 15:14, lgkmcnt in 11:8, expcnt not waited on); then all waves' are.
__device__ __forceinline__ void wait_loads() {
    __builtin_amdgcn_s_waitcnt(0x7 << 4);
#ifdef GSVK_HOSTEMU
    __syncthreads();
#else
    asm volatile("s_barrier" ::: "memory");
#endif
}

// LDS of a workgroup
template <int HD>
struct ChunkLds {
    uint16_t k[2][CH_KEYS * HD];
    uint16_t v[2][CH_KEYS * HD];
    int flag[2];   // [0] a table entry names no page; [1] tile + 1 that holds infinities or NaNs
};

// The key tiles of row tile rt of (s, kvh): the first, and how many (at least one, which may hold
// nothing that is seen)
struct Span { int first, num; };
__device__ __forceinline__ Span span_of(const PagedAttn & a, const Seq & s, int rt) {
    const int r0 = rt * CH_ROWS;
    const int klo = key_lo(a, s, r0 / a.group), khi = key_hi(s, (min(r0 + CH_ROWS, s.rows) - 1) / a.group);
    Span sp;
    sp.first = klo / CH_KEYS;
    sp.num = max(1, (khi + CH_KEYS - 1) / CH_KEYS - sp.first);
    return sp;
}

// Row tile rt of head kvh of sequence s (index b), key tiles [kt0, kt1) of it. part: null where these
// are all of them (the output is final), else where the unnormalised output [CH_ROWS][HD] and (maximum,
// sum) [CH_ROWS][2] go.
template <class T, int HD>
__device__ __forceinline__ void chunk_tile(const PagedAttn & a, const Seq & s, int b, int kvh, int rt, int kt0, int kt1,
                                           float * part, ChunkLds<HD> & lds) {
    constexpr int C = HD / 8, NT = CH_WAVES * 64;
    constexpr int NK = HD / 16, DT = HD / 32;
    constexpr int NL = C / CH_WAVES;   // direct loads of a wave per tile of K (and of V)
    auto & s_k = lds.k;
    auto & s_v = lds.v;
    auto & s_flag = lds.flag;

    const int r0 = rt * CH_ROWS;
    const int tid = threadIdx.x, lane = tid & 63, li = lane & 31, lh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nh = a.group * a.kv.n_kv;
    // the key ranges of the workgroup and of this wave
    const int tokf = r0 / a.group, tokl = (min(r0 + CH_ROWS, s.rows) - 1) / a.group;
    const int klo = key_lo(a, s, tokf), khi = key_hi(s, tokl);
    const int lo_max = key_lo(a, s, tokl), hi_min = key_hi(s, tokf);
    const int rw = r0 + wave * 32;
    const bool idle = rw >= s.rows;
    const int tw0 = min(rw, s.rows - 1) / a.group, tw1 = min(rw + 31, s.rows - 1) / a.group;
    const int wlo_max = key_lo(a, s, tw1), whi_min = key_hi(s, tw0);   // (tiles between are seen whole)
    const int r = min(rw + li, s.rows - 1), tok = r / a.group, h = kvh * a.group + r % a.group;
    const int lo = key_lo(a, s, tok), hi = key_hi(s, tok);

    typename T::v8 qf[NK];
    {
        const uint16_t * qp = a.q + (s.row0 + tok) * a.q_stride + h * HD + 8 * lh;
#pragma unroll
        for (int c = 0; c < NK; c++) qf[c] = v8_of<T>(*reinterpret_cast<const uint4 *>(qp + 16 * c));
    }
    pg_const * tb = (pg_const *) (a.kv.table + b * a.kv.table_stride);

    // A wave's loads of a tile: load j brings the 64 16-byte pieces from piece (j CH_WAVES + wave) * 64 on,
    // all within one group of 16 keys, so within one page.
    const auto piece = [&](int j) { return j * CH_WAVES + wave; };
    uint32_t off_k[NL], off_v[NL];
#pragma unroll
    for (int j = 0; j < NL; j++) {
        const int u = piece(j) * 64 + lane, key = u / C;
        off_k[j] = ((key & 15) * HD + (((u % C) ^ swz_k<HD>(key)) << 3)) * 2;
        off_v[j] = ((key & 15) * HD + (((u % C) ^ swz_vc<HD>(key)) << 3)) * 2;
    }
    // pages of the wave's key groups in tile kt (past the last tile: that tile's), and their byte offsets
    const auto group_of = [&](int kt, int j) {
        return min(kt, kt1 - 1) * CH_KEYS + piece(j) * (CH_KEYS / C) / 16 * 16;
    };
    const auto pages = [&](int kt, int (&pg)[NL]) {
#pragma unroll
        for (int j = 0; j < NL; j++) pg[j] = page_of(a, tb, group_of(kt, j));
    };
    const auto offsets = [&](int kt, const int (&pg)[NL], int64_t (&at)[NL]) {
#pragma unroll
        for (int j = 0; j < NL; j++) at[j] = key_at<HD>(a, pg[j], kvh, group_of(kt, j)) * 2;
    };
    int pg_n[NL] = {};       // pages of the tile whose K comes next: read a step ahead
    int64_t at_v[NL] = {};   // offsets of the tile whose V comes next
    const auto load = [&](const uint16_t * cache, const int64_t (&at)[NL], const uint32_t (&off)[NL], uint16_t * lds) {
#pragma unroll
        for (int j = 0; j < NL; j++) load_lds(reinterpret_cast<const char *>(cache) + at[j], off[j], lds + piece(j) * 512);
    };

    float m = M_NONE, l = 0.0f;
    pg_f16 o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = pg_f16{};

    // operand registers: K of a quarter of the scores' products (k = q / 2), V of the 16 keys 16 q .. + 15
    const auto read_k = [&](uint4 (&kf)[NK / 2], int buf, int q) {
        const int key = 32 * (q >> 1) + li;
#pragma unroll
        for (int i = 0; i < NK / 2; i++) {
            const int c = (q & 1) * (NK / 2) + i;
            kf[i] = *reinterpret_cast<const uint4 *>(&s_k[buf][key * HD + (((2 * c + lh) ^ swz_k<HD>(key)) << 3)]);
        }
    };
    const auto read_v = [&](typename T::v8 (&vf)[DT], int buf, int q) {
        const int key = 16 * q + 4 * lh + ((lane & 15) >> 2);
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const int ch = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
            const uint16_t * p = &s_v[buf][key * HD + ((ch ^ swz_vc<HD>(key)) << 3) + 4 * (lane & 1)];
            const uint16_t * p2 = &s_v[buf][(key + 8) * HD + ((ch ^ swz_vc<HD>(key + 8)) << 3) + 4 * (lane & 1)];
            vf[d] = v8_of<T>(lds_tr4(p), lds_tr4(p2));
        }
    };
    const auto mul_k = [&](pg_f16 (&sc)[2], const uint4 (&kf)[NK / 2], int q) {
#pragma unroll
        for (int i = 0; i < NK / 2; i++) {
            const int c = (q & 1) * (NK / 2) + i;
            sc[q >> 1] = mfma32<T>(v8_of<T>(kf[i]), qf[c], c ? sc[q >> 1] : pg_f16{});
        }
    };
    // S^T of the tile in buffer buf
    const auto scores = [&](pg_f16 (&sc)[2], int buf) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            uint4 kf[NK / 2];
            read_k(kf, buf, q);
            mul_k(sc, kf, q);
        }
    };
    bool has_bad = false;
    // unseen keys of tile kt to -inf
    const auto mask = [&](pg_f16 (&sc)[2], int kt) {
        const int kb = kt * CH_KEYS;
        uint32_t ok = 0xf;
        if (has_bad) {
            ok = 0;
            for (int g = 0; g < CH_KEYS / 16; g++) ok |= (uint32_t) (page_of(a, tb, kb + 16 * g) >= 0) << g;
        }
        const int from = lo - kb - 4 * lh;
        const uint32_t num = (uint32_t) max(hi - lo, 0);
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int v = 0; v < 16; v++) {
                const int j = 32 * k + 8 * (v >> 2) + (v & 3);   // (+ 4 lh)
                if ((uint32_t) (j - from) >= num) sc[k][v] = -INFINITY;
                if ((v & 7) == 7) {
                    if (!((ok >> (2 * k + (v >> 3))) & 1))
#pragma unroll
                        for (int w = v - 7; w <= v; w++) sc[k][w] = -INFINITY;
                    __builtin_amdgcn_sched_barrier(0);   // (otherwise all 32 conditions are held at once)
                }
            }
    };
    const auto top_of = [&](const pg_f16 (&sc)[2]) {
        float top = fmaxf(sc[0][0], sc[1][0]);
#pragma unroll
        for (int v = 1; v < 16; v++) top = fmaxf(fmaxf(top, sc[0][v]), sc[1][v]);
        return top;
    };
    float top = -INFINITY;   // this lane's largest score of the current tile
    // Tile kt: S^T in sc, V in buffer buf; computes S^T of the tile after it from the other buffer.
    // In four stages of 16 keys: a stage's exponentials run while the matrix cores work on a
    // quarter of the next scores and on the weighted sum of the stage before.
    const auto step = [&](int kt, pg_f16 (&sc)[2], pg_f16 (&sn)[2], int buf) {
        const int kb = kt * CH_KEYS;
        if (kb < lo_max || kb + CH_KEYS > hi_min || has_bad) {
            // values that no row sees become zeros; infinities and NaNs are taken out
            for (int u = tid; u < CH_KEYS * C; u += NT) {
                const int key = u / C;
                uint4 * p = reinterpret_cast<uint4 *>(&s_v[buf][u * 8]);
                uint4 x = *p;
                const bool see = kb + key >= klo && kb + key < khi && (!has_bad || page_of(a, tb, kb + key) >= 0);
                if (see && !any_odd<T>(x)) continue;
                if (see) s_flag[1] = kt + 1;
                clear_odd<T>(x);
                *p = see ? x : make_uint4(0, 0, 0, 0);
            }
            __syncthreads();
        }
        // (the first operands are on their way from LDS while the loads are issued)
        uint4 kf[2][NK / 2];
        read_k(kf[0], buf ^ 1, 0);
        // V of the next tile, K of the one after it, into the buffers that the last step read
        if (kt + 1 < kt1) load(a.kv.v, at_v, off_v, s_v[buf ^ 1]);
        if (kt + 2 < kt1) {
            offsets(kt + 2, pg_n, at_v);
            load(a.kv.k, at_v, off_k, s_k[buf]);
            pages(kt + 3, pg_n);
        }
        top *= a.scale_log2;
        if (__any(top > m + M_ROOM)) {
            const float mn = fmaxf(m, max_x32(top) - M_SET);
            const float f = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int v = 0; v < 16; v++) o[d][v] *= f;
        }
        typename T::v8 vf[2][DT], pf;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if (q < 3) read_k(kf[(q + 1) & 1], buf ^ 1, q + 1);
            read_v(vf[q & 1], buf, q);
            mul_k(sn, kf[q & 1], q);
            if (q > 0) {
#pragma unroll
                for (int d = 0; d < DT; d++) o[d] = mfma32<T>(vf[(q - 1) & 1][d], pf, o[d]);
            }
            float p[8], sum = 0.0f;
#pragma unroll
            for (int v = 0; v < 8; v++) {
                p[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[q >> 1][8 * (q & 1) + v], a.scale_log2, -m));
                sum += p[v];
            }
            l += sum;
            asm volatile("" : "+v"(l));   // (summed here: put off, the sum would keep all 32 values live)
            pf = v8_of<T>(make_uint4(pg_pack<T>(p[0], p[1]), pg_pack<T>(p[2], p[3]), pg_pack<T>(p[4], p[5]),
                                     pg_pack<T>(p[6], p[7])));
            // one product at a time among the vector instructions: in order, a run of products
            // would hold up the exponentials behind it
#pragma unroll
            for (int i = 0; i < NK / 2 + (q > 0 ? DT : 0); i++) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                if (q > 0) __builtin_amdgcn_sched_group_barrier(0x402, 28 / (NK / 2 + DT), 0);
                else __builtin_amdgcn_sched_group_barrier(0x402, 28 / (NK / 2), 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] = mfma32<T>(vf[1][d], pf, o[d]);
        if (s_flag[1] == kt + 1) {   // the infinities and NaNs that some of the rows see
            for (int j = 0; j < CH_KEYS; j++) {
                const int key = kb + j, page = page_of(a, tb, key);
                if (page < 0 || key < klo || key >= khi) continue;
                const uint16_t * vp = a.kv.v + key_at<HD>(a, page, kvh, key) + 4 * lh;
                const bool see = key >= lo && key < hi;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int v = 0; v < 16; v++) {
                        const uint16_t u = vp[32 * d + 8 * (v >> 2) + (v & 3)];
                        if (see && is_odd<T>(u)) o[d][v] += T::up(u);
                        if ((v & 3) == 3) __builtin_amdgcn_sched_barrier(0);
                    }
            }
        }
        if (!(kb + CH_KEYS >= wlo_max && kb + 2 * CH_KEYS <= whi_min && !has_bad)) mask(sn, kt + 1);
        top = top_of(sn);
        wait_loads();   // V of the next tile and K of the one after it are there
    };

    {
        if (tid < 2) s_flag[tid] = 0;
        int pg[NL], pg2[NL];
        pages(kt0, pg);
        pages(kt0 + 1, pg2);
        pages(kt0 + 2, pg_n);
        offsets(kt0, pg, at_v);
        load(a.kv.k, at_v, off_k, s_k[0]);
        load(a.kv.v, at_v, off_v, s_v[0]);
        offsets(kt0 + 1, pg2, at_v);
        load(a.kv.k, at_v, off_k, s_k[1]);   // (of a single tile: the same again)
        // table entries that name no page: rare, and every tile then takes its masks
        bool bad = false;
        const int c0 = (kt0 * CH_KEYS) >> a.kv.page_shift, c1 = (min(kt1 * CH_KEYS, khi) - 1) >> a.kv.page_shift;
        for (int c = c0 + tid; c <= c1; c += NT) bad |= page_of(a, tb, c << a.kv.page_shift) < 0;
        wait_loads();
        if (bad) s_flag[0] = 1;
        pg_f16 s0[2], s1[2];
        scores(s0, 0);
        __syncthreads();   // (the flag is set; buffer 0 of K is free)
        has_bad = __builtin_amdgcn_readfirstlane(s_flag[0]) != 0;
        {
            const int kb = kt0 * CH_KEYS;
            if (!(kb >= wlo_max && kb + CH_KEYS <= whi_min && !has_bad)) mask(s0, kt0);
            top = top_of(s0);
        }
        for (int kt = kt0; kt < kt1; kt += 2) {
            step(kt, s0, s1, 0);
            if (kt + 1 < kt1) step(kt + 1, s1, s0, 1);
        }
    }

    if (idle) return;
    l = sum_x32(l);
    const int64_t row = s.row0 + tok, id = row * nh + h;
    const bool valid = rw + li < s.rows;
    if (part) {
        // in register order: 1 KB per store
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int v = 0; v < 16; v += 4)
                *reinterpret_cast<float4 *>(part + (((wave * DT + d) * 4 + v / 4) * 64 + lane) * 4) =
                    make_float4(o[d][v], o[d][v + 1], o[d][v + 2], o[d][v + 3]);
        if (lh == 0) *reinterpret_cast<float2 *>(part + CH_ROWS * HD + 2 * (wave * 32 + li)) = make_float2(m, l);
        return;
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    const auto val = [&](int d, int v) { return l != 0.0f ? o[d][v] * inv : 0.0f; };
    if (a.out_f32) {
        if (valid)
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int v = 0; v < 16; v += 4)
                    *reinterpret_cast<float4 *>((float *) a.out + row * a.out_stride + h * HD + 32 * d + 2 * v + 4 * lh) =
                        make_float4(val(d, v), val(d, v + 1), val(d, v + 2), val(d, v + 3));
    } else {
        // The lane 32 away holds the other 4 of 8 dims: the two trade halves of two groups of 8 and store
        // 16 bytes each.
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int v = 0; v < 16; v += 8) {
                const auto x = __builtin_amdgcn_permlane32_swap(pg_pack<T>(val(d, v), val(d, v + 1)),
                                                                pg_pack<T>(val(d, v + 4), val(d, v + 5)), false, false);
                const auto y = __builtin_amdgcn_permlane32_swap(pg_pack<T>(val(d, v + 2), val(d, v + 3)),
                                                                pg_pack<T>(val(d, v + 6), val(d, v + 7)), false, false);
                if (valid)
                    *reinterpret_cast<uint4 *>((uint16_t *) a.out + row * a.out_stride + h * HD + 32 * d + 2 * v + 8 * lh) =
                        make_uint4(x[0], y[0], x[1], y[1]);
            }
    }
    if (a.lse && lh == 0 && valid) a.lse[id] = lse_of(m, l);
}

// What a launch of chunks holds in LDS: a workgroup past the first a.chunk_groups takes the sequences
// of few rows that stand beside the chunks (no launch of their own: 10 us of a small mixed call).
template <int HD>
union MixLds {
    ChunkLds<HD> chunk;
    FewLds<HD, 2, CH_WAVES> few;
};
template <class T, int HD>
__device__ __forceinline__ void few_beside(const PagedAttn & a, MixLds<HD> & lds) {
    const int f = (int) blockIdx.x - a.chunk_groups, split = f % a.nsplit, kvh = f / a.nsplit % a.kv.n_kv;
    few_tile<T, HD, 2, CH_WAVES>(a, f / a.nsplit / a.kv.n_kv, kvh, 0, split, lds.few);
}

// One row tile per workgroup, all its keys. (head, sequence) fastest, then the row tiles from each
// sequence's last, which sees the most keys, to its first: the longest workgroups start first on
// every XCD (ids go round-robin to the 8 XCDs), and with pairs a multiple of 8 an XCD's L2 holds the
// keys of its own pairs only (8191 tokens, 8 heads of 128: 777 us with the tiles fastest, the CUs busy
// for 0.69 of it; 594 us so). An XCD deals its workgroups to 4 shader engines in turn, so the order of the
// sequences shifts by one every second round: else an engine would get the same sequence, the longest
// perhaps, each time (8 prompts of 700 to 4000, 16 heads over 4 of 128: 423 -> 290 us; 4 of 1428 to 3250, 64 over
// 8: 655 -> 575; 2 of 1200 to 4000: 422 -> 374; a shift every round leaves these 2 as they were).
template <class T, int HD>
__global__ void __launch_bounds__(CH_WAVES * 64, HD == 32 ? 4 : 2) k_attn_paged_chunk(PagedAttn a) {
    __shared__ __align__(16) MixLds<HD> lds;
    if ((int) blockIdx.x >= a.chunk_groups) {
        few_beside<T, HD>(a, lds);
        return;
    }
    const int pairs = a.kv.n_kv * a.kv.B, pair = blockIdx.x % pairs;
    const int kvh = pair % a.kv.n_kv, b = (pair / a.kv.n_kv + (int) (blockIdx.x / pairs) / 2) % a.kv.B;
    const Seq s = seq_of(a, b);
    const int rt = (s.rows + CH_ROWS - 1) / CH_ROWS - 1 - (int) (blockIdx.x / pairs);
    if (rt < 0 || s.rows < a.min_rows) return;
    const Span sp = span_of(a, s, rt);
    chunk_tile<T, HD>(a, s, b, kvh, rt, sp.first, sp.first + sp.num, nullptr, lds.chunk);
}

// Row tiles of unequal length. Every workgroup computes the same list of row tiles and running sums of
// their key tiles, then, by a.ordered,
//   1  takes one whole row tile: the ids go from the longest to the shortest, so that the workgroups that share
//      a CU, and those that come last, are not long ones by chance (of more than BAL_SORT from the list's end
//      to its start, without the sums: the count of longer ones is quadratic, and every CU gets several);
//   0  takes a run of key tiles: those of all row tiles in the order (head, sequence, row tile, key) are
//      cut into equal runs, one per workgroup, and the ids of an XCD take consecutive runs. A row tile that a
//      cut goes through is joined by k_attn_paged_join. For few row tiles over many keys.
constexpr int BAL_GROUPS = 256, BAL_SEQS = 4096, BAL_TILES = 1536, BAL_LEAST = 4, BAL_SORT = 256;

struct BalHead { int64_t run; int tiles, pad; };    // key tiles per workgroup, row tiles of a head
struct BalTile { int first, num, b, rt; };          // a row tile's place in its head's list of key tiles
template <int HD>
constexpr size_t bal_slot() { return (size_t) CH_ROWS * (HD + 2); }   // floats

struct BalLds {
    uint16_t tiles[BAL_SEQS + 1];   // row tiles before each sequence (two workgroups fit a CU's LDS with heads of 128)
    int units[BAL_TILES + 1];   // key tiles before each row tile of a head
    int wave[CH_WAVES];
};

// Exclusive prefix sums of x over the workgroup's threads; total to every thread. Two barriers.
__device__ __forceinline__ int scan_group(int x, int * s_wave, int & total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int y = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int z = __shfl_up(y, d, 64);
        if (lane >= d) y += z;
    }
    if (lane == 63) s_wave[wave] = y;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < CH_WAVES; w++) {
        if (w < wave) before += s_wave[w];
        total += s_wave[w];
    }
    __syncthreads();
    return before + y - x;
}
// the last i in [0, n) with p[i] <= x (p ascending, p[0] <= x)
template <typename I>
__device__ __forceinline__ int last_le(const I * p, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <class T, int HD>
__global__ void __launch_bounds__(CH_WAVES * 64, 2) k_attn_paged_balanced(PagedAttn a) {
    __shared__ __align__(16) MixLds<HD> lds;
    __shared__ BalLds bal;
    if ((int) blockIdx.x >= a.chunk_groups) {
        few_beside<T, HD>(a, lds);
        return;
    }
    const int tid = threadIdx.x;
    // row tiles of the sequences
    int tiles = 0;
    for (int b0 = 0; b0 < a.kv.B; b0 += CH_WAVES * 64) {
        int n = 0, add = 0;
        const int b = b0 + tid;
        if (b < a.kv.B) {
            const Seq s = seq_of(a, b);
            if (s.rows >= a.min_rows) n = min((s.rows + CH_ROWS - 1) / CH_ROWS, a.bal_most);
        }
        n = scan_group(n, bal.wave, add);
        if (b < a.kv.B) bal.tiles[b] = (uint16_t) min(tiles + n, 0xffff);
        tiles = min(tiles + add, 0xffff);
    }
    if (tid == 0) bal.tiles[a.kv.B] = (uint16_t) tiles;
    __syncthreads();
    tiles = __builtin_amdgcn_readfirstlane(min(tiles, a.bal_most));   // (more only if seq_start does not ascend)
    if (tiles == 0) {
        if (blockIdx.x == 0 && tid == 0 && !a.ordered) *a.bal_head = BalHead{1, 0, 0};
        return;
    }
    int units = 0;   // key tiles of a head
    const int summed = !a.ordered || tiles <= BAL_SORT ? tiles : 0;
    for (int e0 = 0; e0 < summed; e0 += CH_WAVES * 64) {
        int n = 0, add = 0;
        const int e = e0 + tid;
        if (e < summed) {
            const int b = last_le(bal.tiles, a.kv.B, e);
            n = span_of(a, seq_of(a, b), e - bal.tiles[b]).num;
        }
        n = scan_group(n, bal.wave, add);
        if (e < summed) bal.units[e] = units + n;
        units += add;
    }
    if (tid == 0) bal.units[summed] = units;
    __syncthreads();
    units = __builtin_amdgcn_readfirstlane(units);
    if (a.ordered) {
        // heads fastest: an XCD keeps its heads
        const int rank = (int) blockIdx.x / a.kv.n_kv, kvh = (int) blockIdx.x % a.kv.n_kv;
        if (rank >= tiles) return;
        int e = tiles - 1 - rank;
        if (tiles <= BAL_SORT) {
            if (tid < tiles) {
                const int n = bal.units[tid + 1] - bal.units[tid];
                int r = 0;
                for (int i = 0; i < tiles; i++) {
                    const int x = bal.units[i + 1] - bal.units[i];
                    r += x > n || (x == n && i < tid);
                }
                if (r == rank) bal.wave[0] = tid;
            }
            __syncthreads();
            e = __builtin_amdgcn_readfirstlane(bal.wave[0]);
        }
        const int b = __builtin_amdgcn_readfirstlane(last_le(bal.tiles, a.kv.B, e));
        const int rt = e - __builtin_amdgcn_readfirstlane((int) bal.tiles[b]);
        const Seq s = seq_of(a, b);
        const Span sp = span_of(a, s, rt);
        chunk_tile<T, HD>(a, s, b, kvh, rt, sp.first, sp.first + sp.num, nullptr, lds.chunk);
        return;
    }
    const int64_t total = (int64_t) units * a.kv.n_kv;
    const int64_t share = (total + BAL_GROUPS - 1) / BAL_GROUPS;
    const int64_t run = max(share, (int64_t) min(BAL_LEAST, (units + tiles - 1) / tiles));
    if (blockIdx.x == 0 && tid == 0) *a.bal_head = BalHead{run, tiles, 0};

    const int w = (int) (blockIdx.x % 8) * (BAL_GROUPS / 8) + (int) (blockIdx.x / 8);
    const int64_t u0 = w * run, u1 = min(total, u0 + run);
    if (u0 >= u1) return;
    // (the values below are uniform; said so for the direct loads, whose base is scalar)
    int kvh = __builtin_amdgcn_readfirstlane((int) (u0 / units));
    const int at = __builtin_amdgcn_readfirstlane((int) (u0 - (int64_t) kvh * units));
    int e = __builtin_amdgcn_readfirstlane(last_le(bal.units, tiles, at));
    int b = __builtin_amdgcn_readfirstlane(last_le(bal.tiles, a.kv.B, e));
    int64_t left = u1 - u0;
    int t0 = at - __builtin_amdgcn_readfirstlane(bal.units[e]);
    Seq s = seq_of(a, b);
    for (bool more = false;; more = true) {
        const int first = __builtin_amdgcn_readfirstlane(bal.units[e]);
        const int num = __builtin_amdgcn_readfirstlane(bal.units[e + 1]) - first;
        const int t1 = (int) min((int64_t) num, t0 + left);
        const int rt = e - __builtin_amdgcn_readfirstlane((int) bal.tiles[b]);
        const Span sp = span_of(a, s, rt);
        float * part = nullptr;
        if (t1 - t0 < num) part = a.bal_part + (int64_t) (2 * w + more) * bal_slot<HD>();
        if (t0 == 0 && tid == 0) a.bal_tiles[kvh * tiles + e] = BalTile{first, num, b, rt};
        chunk_tile<T, HD>(a, s, b, kvh, rt, sp.first + t0, sp.first + t1, part, lds.chunk);
        left -= t1 - t0;
        if (left == 0) break;
        t0 = 0;
        if (++e == tiles) {
            e = 0;
            kvh++;
        }
        const int next = __builtin_amdgcn_readfirstlane(last_le(bal.tiles, a.kv.B, e));
        if (next != b) {
            b = next;
            s = seq_of(a, b);
        }
    }
}

// A row tile e of head kvh, if k_attn_paged_balanced has cut it: part x of it (a wave's 32 rows and 32
// dims), a thread 4 dims of a row, as the wave stored them
template <class T, int HD>
__device__ __forceinline__ void join_tile(const PagedAttn & a, int e, int kvh, int x0) {
    constexpr int DT = HD / 32;
    const BalHead hd = *a.bal_head;
    if (e >= hd.tiles) return;
    const BalTile t = a.bal_tiles[kvh * hd.tiles + e];
    // (a head's key tiles follow the last head's)
    const BalTile last = a.bal_tiles[hd.tiles - 1];
    const int64_t u0 = (int64_t) kvh * (last.first + last.num) + t.first, u1 = u0 + t.num;
    const int w0 = (int) (u0 / hd.run), w1 = (int) ((u1 - 1) / hd.run);
    if (w0 == w1) return;
    const Seq s = seq_of(a, t.b);
    const int lane = threadIdx.x & 63, vq = threadIdx.x >> 6;
    const int rl = x0 / DT * 32 + (lane & 31), r = t.rt * CH_ROWS + rl;
    if (r >= s.rows) return;
    const bool late = w0 * hd.run < u0;   // the first part is not its workgroup's first
    float M = M_NONE, L = 0.0f, x[4] = {};
    for (int w = w0; w <= w1; w += 4) {   // (four parts' loads in flight)
        float2 ml[4];
        float4 u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int wi = min(w + i, w1);
            const float * part = a.bal_part + (2 * (int64_t) wi + (wi == w0 && late)) * bal_slot<HD>();
            ml[i] = *reinterpret_cast<const float2 *>(part + CH_ROWS * HD + 2 * rl);
            u[i] = *reinterpret_cast<const float4 *>(part + ((x0 * 4 + vq) * 64 + lane) * 4);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (w + i > w1) break;
            const float mn = fmaxf(M, ml[i].x), c = __builtin_amdgcn_exp2f(M - mn), f = __builtin_amdgcn_exp2f(ml[i].x - mn);
            M = mn;
            L = __builtin_fmaf(L, c, ml[i].y * f);
            x[0] = __builtin_fmaf(x[0], c, u[i].x * f); x[1] = __builtin_fmaf(x[1], c, u[i].y * f);
            x[2] = __builtin_fmaf(x[2], c, u[i].z * f); x[3] = __builtin_fmaf(x[3], c, u[i].w * f);
        }
    }
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = L != 0.0f ? x[i] * inv : 0.0f;
    const int tok = r / a.group, h = kvh * a.group + r % a.group, col = x0 % DT * 32 + 8 * vq + 4 * (lane >> 5);
    store4<T>(a, s.row0 + tok, h * HD + col, x[0], x[1], x[2], x[3]);
    if (a.lse && col == 0) a.lse[(s.row0 + tok) * a.group * a.kv.n_kv + h] = lse_of(M, L);
}

// ---- joining the splits ------------------------------------------------------------------------------

// A workgroup takes 256 / (HD / 8) / SL rows of (head kvh, sequence b), the x0-th such group; a row's
// splits are dealt to SL groups of HD / 8 threads, which hold 8 dims each, and the groups are joined
// through LDS. SL 16 where there are more than 4 splits (64 splits of 2 x 64 rows of 128: 54.7 us with SL 1,
// one split after another; 5.6 us so).
template <int HD, int SL>
struct MergeLds {
    float x[256 / (HD / 8) / SL][SL][HD + 4];
    float ml[256 / (HD / 8) / SL][SL][2];
};
template <class T, int HD, int SL>
__device__ __forceinline__ void merge_rows(const PagedAttn & a, int b, int kvh, int x0, MergeLds<HD, SL> & lds) {
    constexpr int C = HD / 8, R = 256 / C / SL;
    auto & s_x = lds.x;
    auto & s_ml = lds.ml;
    const Seq s = seq_of(a, b);
    const int r0 = x0 * R;
    if (r0 >= s.rows || s.rows > FEW_ROWS) return;
    const int rr = threadIdx.x / (C * SL), sl = threadIdx.x / C % SL, col = (threadIdx.x % C) * 8;
    const int r = min(r0 + rr, s.rows - 1);
    const int nh = a.group * a.kv.n_kv, tok = r / a.group, h = kvh * a.group + r % a.group;
    const int64_t row = s.row0 + tok, id = row * nh + h, step = a.kv.tokens * nh;
    float M = M_NONE, L = 0.0f, x[8] = {};
    for (int i = sl; i < a.nsplit; i += SL) {
        const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + 2 * (i * step + id));
        const float4 * p = reinterpret_cast<const float4 *>(a.part_o + (i * step + id) * HD + col);
        const float4 u = p[0], w = p[1];
        const float mn = fmaxf(M, ml.x), e = __builtin_amdgcn_exp2f(M - mn), f = __builtin_amdgcn_exp2f(ml.x - mn);
        M = mn;
        L = __builtin_fmaf(L, e, ml.y * f);
        x[0] = __builtin_fmaf(x[0], e, u.x * f); x[1] = __builtin_fmaf(x[1], e, u.y * f);
        x[2] = __builtin_fmaf(x[2], e, u.z * f); x[3] = __builtin_fmaf(x[3], e, u.w * f);
        x[4] = __builtin_fmaf(x[4], e, w.x * f); x[5] = __builtin_fmaf(x[5], e, w.y * f);
        x[6] = __builtin_fmaf(x[6], e, w.z * f); x[7] = __builtin_fmaf(x[7], e, w.w * f);
    }
    if constexpr (SL > 1) {
        if (col == 0) {
            s_ml[rr][sl][0] = M;
            s_ml[rr][sl][1] = L;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) s_x[rr][sl][col + i] = x[i];
        __syncthreads();
        if (sl) return;
        for (int i = 0; i < SL; i++) M = fmaxf(M, s_ml[rr][i][0]);
        L = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < SL; k++) {
            const float f = __builtin_amdgcn_exp2f(s_ml[rr][k][0] - M);
            L = __builtin_fmaf(s_ml[rr][k][1], f, L);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = __builtin_fmaf(s_x[rr][k][col + i], f, x[i]);
        }
    }
    if (r0 + rr >= s.rows) return;
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = L != 0.0f ? x[i] * inv : 0.0f;
    store8<T>(a, row, h * HD + col, x);
    if (a.lse && col == 0) a.lse[id] = lse_of(M, L);
}

// Joins what the launch before it has cut: first the row tiles of chunks, then the rows of few
template <class T, int HD, int SL>
__global__ void __launch_bounds__(256) k_attn_paged_join(PagedAttn a) {
    __shared__ MergeLds<HD, SL> lds;
    constexpr int X = CH_WAVES * (HD / 32), R = 256 / (HD / 8) / SL;
    const int tiles = a.ordered ? 0 : a.bal_most * a.kv.n_kv * X;
    int i = blockIdx.x;
    if (i < tiles) {
        join_tile<T, HD>(a, i / X % a.bal_most, i / X / a.bal_most, i % X);
        return;
    }
    i -= tiles;
    const int per = (a.few_rows + R - 1) / R;
    merge_rows<T, HD, SL>(a, i / per / a.kv.n_kv, i / per % a.kv.n_kv, i % per, lds);
}

// ---- the host's side -----------------------------------------------------------------------------------

// How a call is cut: a function of its arguments alone (the workspace's size follows from it)
struct Plan {
    bool few, chunk;       // sequences of few rows can be there; chunks can
    int few_rows, few_qt, few_waves, few_tiles, few_split;
    int chunk_tiles;       // row tiles of the longest sequence
    int deal;              // of chunks to workgroups (Deal)
    int most_tiles;        // with lists: the most row tiles that there can be per head
};

// How chunks are dealt to workgroups, by estimated times in us. A step of 64 keys takes `step` with one
// workgroup on a CU, and the chip as a whole `share` of that per CU with two (small heads leave one waiting
// for its own exponentials). One row tile per workgroup takes the longest row tile's
// steps or the chip's share of all; in the order of the grid two long ones can share a CU while the
// chip holds about all of them (512 workgroups), by length they do not, at the price of the list. Equal
// runs, one workgroup on a CU, take 1.4 of the share and a fixed cost that grows with the partial results. `all` takes the other
// sequences of a batch as 0.7 of the longest. Measured (us; grid order / by length / runs), heads of 128,
// 32 over 8: 4 x 512 tokens over 1000 to 8100 keys 237 / 220 / 289, two chunks of 700 to 1000 over 200 to
// 4900 beside 22 single tokens 159 / 149 / 196, 3 prompts of 300 to 2500 72 / 80 / 185, one of 2000 54 / 59 / 140,
// 6 x 100 to 700 over up to 3700 129 / 104 / 190, 2 x 256 over 2900 69 / 74 / 53, 64 over 8000 158 / 165 / 36;
// 5 over 1, 4 x 100 over 7000 to 11000 beside 3 single tokens 210 / 216 / 42; heads of 64: 8 x 200 to 800 over up
// to 3800, 16 over 8 70 / 59 / 101; heads of 32: 2 x 125 to 307 over 4600, 64 over 8 59 / 61 / 52.
enum Deal { DEAL_GRID, DEAL_LENGTH, DEAL_RUNS };
Deal deal_of(int B, int hd, double tiles, double groups, double keys, double mean_keys, int64_t most) {
    const double step = hd == 128 ? 1.0 : hd == 64 ? 0.75 : 0.7, share = hd == 128 ? 1.0 : hd == 64 ? 0.6 : 0.45;
    const double load = tiles / 256;
    const double longest = keys / 64, mean = mean_keys / 64;
    // (prompts from the start come by length in the grid's order too, once there are more than fit)
    const double old = mean / std::max(longest, 1.0), shared = std::min({load - 1.0, 1.0, old > 0.7 ? 1.0 : 3.0 - load});
    const double slow = 1.1 * (1.0 + std::max(shared, 0.0) * old);
    const double all = mean * tiles / 512 * 1.95 * share * (B > 1 ? 0.7 : 1.0);
    // (a workgroup of the grid beyond a sequence's rows costs its start: a chunk of 4096 tokens beside 255 single
    // ones, 32 over 8 of 128, 937 us of which 0.6 ms are such workgroups; from the list 361)
    const double grid = std::max(longest * slow * step, all) + (groups - tiles) / 512;
    // (one sequence's go well as they are; not put in order the list's end is worse than the grid's, 605 to 575)
    double length = std::max(1.1 * longest * step, most > BAL_SORT ? 1.1 * all : all) + 6 + B / 512.0;
    if (B == 1 || B > BAL_SEQS || most > UINT16_MAX) length = 1e30;
    double runs = 1.4 * all + 22 + 30 * std::min(1.0, tiles / 512) * hd / 128;
    if (B > BAL_SEQS || most > BAL_TILES) runs = 1e30;
    if (grid <= std::min(length, runs)) return DEAL_GRID;
    return length <= runs ? DEAL_LENGTH : DEAL_RUNS;
}

Plan plan_of(int B, int n_kv, int hd, int group, int64_t tokens, int max_new, int64_t max_keys, int window) {
    Plan p{};
    if (max_new > tokens) max_new = (int) tokens;
    max_keys = std::min<int64_t>(max_keys, PG_MAX_KEYS);
    // the most keys of a row tile (of `some` rows): a window's and its own tokens'
    const auto seen = [&](int64_t some) {
        return window ? std::min(max_keys, window + std::min<int64_t>(max_new, some / group + 1)) : max_keys;
    };
    const int64_t rows = (int64_t) max_new * group;
    p.chunk = rows > FEW_ROWS;
    p.few = !p.chunk || (B > 1 && group <= FEW_ROWS);
    if (p.few) {
        p.few_rows = (int) std::min<int64_t>(rows, FEW_ROWS);
        p.few_qt = p.few_rows <= 16 && !p.chunk ? 1 : 2;
        p.few_tiles = (p.few_rows + 16 * p.few_qt - 1) / (16 * p.few_qt);
        const int64_t pairs = (int64_t) B * n_kv;
        p.few_waves = !p.chunk && pairs * p.few_tiles <= 256 ? 8 : 4;
        // A workgroup alone on its CU takes 6 us and 9 us per 1000 keys of 128 (a CU's own bandwidth), so keys are
        // split as far as the CUs go, but not below 128 keys, and only where that gains more than the second launch
        // that joins them costs (5 us; 1 / 2 / 4 / 8 / 16 / 32 splits, us: one sequence of 8 heads of 128 over 2000
        // keys 24 / 18 / 14 / 12 / 10 / 10, 4 over 5000 48 / 31 / 22 / 20 / 25 / 31, 16 over 4000 53 / 41 / 43 / 50 /
        // 64 / 87, 32 over 12000 190 / 200 / 195 / 192 / 228 / 290). With more pairs than CUs workgroups have 4 waves,
        // and are split up to about 16 waves per CU, to no less than 1024 keys (40 sequences of 8 heads of 128 over
        // 12000 keys, 1 / 2 / 4: 269 / 227 / 216); beside chunks they have 4 waves too.
        const int64_t keys = seen(FEW_ROWS), groups = pairs * p.few_tiles;
        int64_t n = std::min(256 / groups, keys / 128);
        if (n > 1 && keys * hd * (n - 1) / n <= 72 * 1024) n = 1;
        if (!p.chunk && p.few_waves == 4) n = std::min((1024 + pairs - 1) / pairs, keys / 1024);
        p.few_split = (int) std::max<int64_t>(1, std::min<int64_t>(n, 64));
        // (chunks of max_new tokens each, unless rows are padding: no launch to join what is hardly there)
        if (p.chunk && tokens >= (int64_t) B * max_new) p.few_split = 1;
    }
    if (p.chunk) {
        p.chunk_tiles = (int) ((rows + CH_ROWS - 1) / CH_ROWS);
        // row tiles of a head: at most one per CH_ROWS rows and one begun per sequence that has more than few
        const int64_t least = std::max<int64_t>(1, tokens * group / CH_ROWS);
        const int64_t most = tokens * group / CH_ROWS + (p.few ? std::min<int64_t>(B, tokens * group / (FEW_ROWS + 1)) : B);
        const double keys = (double) seen(CH_ROWS), mean = std::min(keys, std::max(0.0, (double) max_keys - 0.5 * max_new));
        p.deal = deal_of(B, hd, (double) (least * n_kv), (double) p.chunk_tiles * n_kv * B, keys, mean, most);
        if (p.deal != DEAL_GRID) p.most_tiles = (int) most;
    }
    return p;
}

// The workspace: tables and slots of k_attn_paged_balanced, then the outputs, then the (maximum, sum) of
// the splits of few rows
struct Space { size_t slots, few, ml, end; };
Space space_of(const Plan & p, int64_t rows, int n_kv, int hd) {
    Space w{};
    if (p.deal == DEAL_RUNS) {
        w.slots = (sizeof(BalHead) + (size_t) p.most_tiles * n_kv * sizeof(BalTile) + 255) / 256 * 256;
        w.few = w.slots + 2 * (size_t) BAL_GROUPS * CH_ROWS * (size_t) (hd + 2) * sizeof(float);
    }
    w.ml = w.end = w.few;
    if (p.few_split > 1) {
        w.ml = w.few + (size_t) p.few_split * (size_t) rows * (size_t) hd * sizeof(float);
        w.end = w.ml + (size_t) p.few_split * (size_t) rows * 2 * sizeof(float);
    }
    return w;
}

int64_t chunk_groups_of(const Plan & p, int B, int n_kv) {   // workgroups of chunks
    if (!p.chunk) return 0;
    return p.deal == DEAL_RUNS ? BAL_GROUPS : (int64_t) (p.deal == DEAL_LENGTH ? p.most_tiles : (int64_t) p.chunk_tiles * B) * n_kv;
}
int64_t groups_of(const Plan & p, int B, int n_kv) {   // workgroups of the first launch
    const int64_t few = (int64_t) p.few_tiles * p.few_split * n_kv * B;
    return chunk_groups_of(p, B, n_kv) + few;
}

// rows of few rows that a workgroup of k_attn_paged_join takes, and its workgroups
int join_rows(const Plan & p, int hd) { return 256 / (hd / 8) / (p.few_split > 4 ? 16 : 1); }
int64_t join_groups_of(const Plan & p, int B, int n_kv, int hd) {
    const int64_t per = p.few_split > 1 ? (p.few_rows + join_rows(p, hd) - 1) / join_rows(p, hd) : 0;
    return (p.deal == DEAL_RUNS ? (int64_t) p.most_tiles * n_kv * (CH_WAVES * (hd / 32)) : 0) + per * n_kv * B;
}

template <class T, int HD>
void launch_attn(PagedAttn a, const Plan & p, void * ws, hipStream_t st) {
    const unsigned nkv = (unsigned) a.kv.n_kv, B = (unsigned) a.kv.B;
    const Space w = space_of(p, a.kv.tokens * a.group * a.kv.n_kv, a.kv.n_kv, HD);
    a.bal_head = (BalHead *) ws;
    a.bal_tiles = (BalTile *) (a.bal_head + 1);
    a.bal_part = (float *) ((char *) ws + w.slots);
    a.part_o = (float *) ((char *) ws + w.few);
    a.part_ml = (float *) ((char *) ws + w.ml);
    a.nsplit = p.few ? p.few_split : 1;
    a.few_rows = p.few_rows;
    if (p.chunk) {
        a.min_rows = p.few ? FEW_ROWS + 1 : 1;
        a.bal_most = p.most_tiles;
        a.ordered = p.deal == DEAL_LENGTH;
        a.chunk_groups = (int) chunk_groups_of(p, a.kv.B, a.kv.n_kv);
        const dim3 grid((unsigned) groups_of(p, a.kv.B, a.kv.n_kv)), block(CH_WAVES * 64);
        if (p.deal != DEAL_GRID) hipLaunchKernelGGL((k_attn_paged_balanced<T, HD>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((k_attn_paged_chunk<T, HD>), grid, block, 0, st, a);
    } else {
        const dim3 grid((unsigned) (p.few_tiles * p.few_split), nkv, B), block((unsigned) p.few_waves * 64);
        if (p.few_qt == 1 && p.few_waves == 4) hipLaunchKernelGGL((k_attn_paged_few<T, HD, 1, 4>), grid, block, 0, st, a);
        else if (p.few_qt == 1) hipLaunchKernelGGL((k_attn_paged_few<T, HD, 1, 8>), grid, block, 0, st, a);
        else if (p.few_waves == 4) hipLaunchKernelGGL((k_attn_paged_few<T, HD, 2, 4>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((k_attn_paged_few<T, HD, 2, 8>), grid, block, 0, st, a);
    }
    const int64_t n = join_groups_of(p, a.kv.B, a.kv.n_kv, HD);
    if (n == 0) return;
    if (a.nsplit <= 4) hipLaunchKernelGGL((k_attn_paged_join<T, HD, 1>), dim3((unsigned) n), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_attn_paged_join<T, HD, 16>), dim3((unsigned) n), dim3(256), 0, st, a);
}

template <class T>
void launch_attn(const PagedAttn & a, int hd, const Plan & p, void * ws, hipStream_t st) {
    if (hd == 32) launch_attn<T, 32>(a, p, ws, st);
    else if (hd == 64) launch_attn<T, 64>(a, p, ws, st);
    else launch_attn<T, 128>(a, p, ws, st);
}

bool attn_args(const gsvk_paged_kv * kv, int64_t tokens, int nh, int max_new, int64_t max_keys) {
    return nh >= 1 && nh <= 65535 && kv->n_kv >= 1 && nh % kv->n_kv == 0 && max_new >= 0 && max_keys >= 0
           && tokens >= 0 && tokens * nh <= INT32_MAX;
}

}  // namespace
}  // namespace gsvk

extern "C" size_t gsvk_attn_paged_workspace_bytes(const gsvk_paged_kv * kv, int64_t tokens, int nh, int max_new,
                                                  int64_t max_keys, int window) {
    using namespace gsvk;
    if (!kv || !attn_args(kv, tokens, nh, max_new, max_keys) || kv->B < 1 || tokens == 0 || max_new == 0
        || window < 0) return 0;
    if (kv->hd != 32 && kv->hd != 64 && kv->hd != 128) return 0;
    return space_of(plan_of(kv->B, kv->n_kv, kv->hd, nh / kv->n_kv, tokens, max_new, max_keys, window), tokens * nh, kv->n_kv, kv->hd).end;
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
    GSVK_REQUIRE(window >= 0 && max_new >= 0 && max_keys >= 0, "attn_paged: window, max_new and max_keys must not be negative");
    GSVK_REQUIRE(attn_args(kv, tokens, nh, max_new, max_keys), "attn_paged: tokens * nh must be below 2^31");
    GSVK_REQUIRE(out_type == GSVK_TYPE_F32 || out_type == kv->type,
                 "attn_paged: out_type %d is neither F32 nor the cache's type", out_type);
    GSVK_REQUIRE(scale > 0.0f && std::isfinite(scale * 1.4426950408889634f), "attn_paged: scale must be positive and finite");
    if (tokens == 0 || kv->B == 0 || max_new == 0) return GSVK_OK;
    GSVK_REQUIRE(q && out, "attn_paged: q and out must be given");
    const int64_t w = (int64_t) nh * kv->hd;
    GSVK_REQUIRE((q_stride >= w && out_stride >= w) || tokens == 1, "attn_paged: a stride is smaller than its row");
    GSVK_REQUIRE((((uintptr_t) q | (uintptr_t) out) & 15) == 0 && q_stride % 8 == 0
                     && out_stride % (out_type == GSVK_TYPE_F32 ? 4 : 8) == 0,
                 "attn_paged: the rows of q and out must be 16-byte aligned");
    const int group = nh / kv->n_kv;
    const Plan p = plan_of(kv->B, kv->n_kv, kv->hd, group, tokens, max_new, max_keys, window);
    const size_t need = space_of(p, tokens * nh, kv->n_kv, kv->hd).end;
    GSVK_REQUIRE(need == 0 || (ws && ws_bytes >= need && ((uintptr_t) ws & 15) == 0),
                 "attn_paged: a workspace of %zu bytes, 16-byte aligned, is needed (%zu given)", need, ws_bytes);
    // (a launch has fewer than 2^32 threads)
    constexpr int64_t MOST = UINT32_MAX / 256;
    GSVK_REQUIRE(groups_of(p, kv->B, kv->n_kv) <= MOST && join_groups_of(p, kv->B, kv->n_kv, kv->hd) <= MOST,
                 "attn_paged: too many row tiles for one launch");
    a.q = (const uint16_t *) q;
    a.q_stride = q_stride;
    a.out = out;
    a.out_stride = out_stride;
    a.lse = lse;
    a.prefix = prefix;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.group = group;
    a.window = window;
    a.max_new = max_new < tokens ? max_new : (int) tokens;
    a.out_f32 = out_type == GSVK_TYPE_F32;
    if (kv->type == GSVK_TYPE_F16) launch_attn<PgF16>(a, kv->hd, p, ws, (hipStream_t) stream);
    else launch_attn<PgBF16>(a, kv->hd, p, ws, (hipStream_t) stream);
    GSVK_LAUNCH_CHECK();
    return GSVK_OK;
}
