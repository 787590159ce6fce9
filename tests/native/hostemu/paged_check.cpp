// Host check of the paged-cache operators (paged_append.hip, paged_attn.hip) compiled for the CPU
// (hip/hip_runtime.h, emu.h) under AddressSanitizer, every buffer of exactly the size that the
// interface asks for: a batch is appended (rotated) to pages and attended to. No access may leave a
// buffer, stale slots (NaN) and unseen keys may not reach an output, and the outputs are those of a
// double-precision evaluation. Test infrastructure only.
//
//   paged_check hd bf16 nh nkv page window prefix f32 poison tail new:keys [new:keys ...]
//
// prefix: 0, or the bidirectional prefix of every sequence; poison 1: the value and key of each
// chunk's last token are NaN, 2: one table entry in seven names no page, 3: seq_start and kv_len are not
// what they should be (rows of several sequences, past the last row, descending; only bounds are checked).
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <string>
#include <vector>

#include "common.h"

namespace gsvk {
static std::string g_err;
void set_error(const char * fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    g_err = buf;
}
const char * get_error() { return g_err.c_str(); }
}  // namespace gsvk

static uint16_t to_bf(float f) {
    uint32_t u;
    std::memcpy(&u, &f, 4);
    if (f != f) return 0x7fc0;
    return (uint16_t) ((u + 0x7fff + ((u >> 16) & 1)) >> 16);
}
// (the host's conversion of fp32 to bf16 is a call of the compiler's runtime library, which not every
// host has; a _Float16 returns in the same register)
extern "C" __attribute__((weak)) _Float16 emu_truncsfbf2(float f) asm("__truncsfbf2");
extern "C" _Float16 emu_truncsfbf2(float f) { return __builtin_bit_cast(_Float16, to_bf(f)); }

static bool g_bf;
static uint16_t enc(float f) { return g_bf ? to_bf(f) : __builtin_bit_cast(uint16_t, (_Float16) f); }
static double dec(uint16_t u) {
    if (!g_bf) return (double) __builtin_bit_cast(_Float16, u);
    return __builtin_bit_cast(float, (uint32_t) u << 16);
}

template <typename T>
static T * buf(size_t n) { return (T *) std::malloc(n * sizeof(T)); }

int main(int argc, char ** argv) {
    if (argc < 12) return 2;
    const int hd = std::atoi(argv[1]), nh = std::atoi(argv[3]), nkv = std::atoi(argv[4]), page = std::atoi(argv[5]);
    const int window = std::atoi(argv[6]), prefix = std::atoi(argv[7]), f32 = std::atoi(argv[8]);
    const int poison = std::atoi(argv[9]), tail = std::atoi(argv[10]);
    g_bf = std::atoi(argv[2]) != 0;
    std::vector<int> n, tot;
    for (int i = 11; i < argc; i++) {
        int x, y;
        if (std::sscanf(argv[i], "%d:%d", &x, &y) != 2) return 2;
        n.push_back(x);
        tot.push_back(y);
    }
    const int B = (int) n.size(), G = nh / nkv;
    int cols = 1, pages = 0, T = 0, max_new = 1, max_keys = 1;
    for (int b = 0; b < B; b++) {
        const int c = (tot[b] + page - 1) / page;
        cols = std::max(cols, c);
        pages += c;
        T += n[b];
        max_new = std::max(max_new, n[b]);
        max_keys = std::max(max_keys, tot[b]);
    }
    const int tokens = T + tail, ps = nkv * page * hd;
    std::mt19937 rng(hd + nh + T);
    std::normal_distribution<float> nd(0.0f, 1.0f);
    std::vector<int> order(pages);
    for (int i = 0; i < pages; i++) order[i] = i;
    std::shuffle(order.begin(), order.end(), rng);
    int32_t * table = buf<int32_t>((size_t) B * cols), * ss = buf<int32_t>(B + 1), * len = buf<int32_t>(B), * pre = buf<int32_t>(B);
    for (int b = 0, at = 0, row = 0; b < B; b++) {
        for (int c = 0; c < cols; c++) table[b * cols + c] = c * page < tot[b] ? order[at++] : 0x7fffffff;
        ss[b] = row;
        ss[b + 1] = row += n[b];
        len[b] = tot[b];
        pre[b] = prefix;
    }
    if (poison == 2)
        for (int i = 0; i < B * cols; i += 7) table[i] = i % 2 ? -1 : pages;
    uint16_t * kc = buf<uint16_t>((size_t) pages * ps), * vc = buf<uint16_t>((size_t) pages * ps);
    const uint16_t nan = enc(NAN);
    for (size_t i = 0; i < (size_t) pages * ps; i++) kc[i] = vc[i] = nan;
    const auto slot = [&](int b, int h, int j) -> int64_t {
        const int pg = j / page < cols ? table[b * cols + j / page] : -1;
        return pg < 0 || pg >= pages ? -1 : (int64_t) pg * ps + ((int64_t) h * page + j % page) * hd;
    };
    for (int b = 0; b < B; b++)
        for (int j = 0; j < tot[b] - n[b]; j++)
            for (int h = 0; h < nkv; h++)
                if (slot(b, h, j) >= 0)
                    for (int d = 0; d < hd; d++) {
                        kc[slot(b, h, j) + d] = enc(nd(rng));
                        vc[slot(b, h, j) + d] = enc(nd(rng));
                    }
    // the new tokens: fp32 rows of a projection
    const int w = (nh + 2 * nkv) * hd, rot = hd / 2, half = rot / 2;
    float * qkv = buf<float>((size_t) tokens * w), * cs = buf<float>((size_t) max_keys * half), * sn = buf<float>((size_t) max_keys * half);
    for (size_t i = 0; i < (size_t) tokens * w; i++) qkv[i] = nd(rng);
    for (int p = 0; p < max_keys; p++)
        for (int i = 0; i < half; i++) {
            cs[p * half + i] = (float) std::cos(p * std::pow(1e4, -(double) i / half));
            sn[p * half + i] = (float) std::sin(p * std::pow(1e4, -(double) i / half));
        }
    if (poison == 1)
        for (int b = 0; b < B; b++)
            if (n[b] > 1)
                for (int d = nh * hd; d < w; d++) qkv[(size_t) (ss[b + 1] - 1) * w + d] = NAN;
    if (poison == 3)
        for (int b = 0; b <= B; b++) {
            ss[b] = b % 3 == 0 ? 0 : b % 3 == 1 ? tokens : 0x7fffffff;
            if (b < B) len[b] = b % 4 == 3 ? -0x7fffffff : b % 4 == 2 ? 0x7fffffff : tot[b];
        }
    gsvk_paged_kv kv{kc, vc, g_bf ? GSVK_TYPE_BF16 : GSVK_TYPE_F16, nkv, hd, page, pages, 0, table, cols, cols, B, ss, len};
    gsvk_rope rope{cs, sn, max_keys, rot, 0, nullptr};
    uint16_t * q = buf<uint16_t>((size_t) tokens * nh * hd);
    for (size_t i = 0; i < (size_t) tokens * nh * hd; i++) q[i] = enc(3.0f);
    int32_t bad = 0;
    if (gsvk_op_paged_append(&kv, qkv, qkv + nh * hd, qkv + (nh + nkv) * hd, GSVK_TYPE_F32, tokens, nh, w, w, w, &rope, q, &bad, nullptr)) {
        std::fprintf(stderr, "%s\n", gsvk::get_error());
        return 1;
    }
    for (int b = 0; b < B && poison != 3; b++)
        for (int i = 0; i < n[b]; i++)
            for (int h = 0; h < nh + nkv; h++) {
                const int p = tot[b] - n[b] + i;
                const float * x = qkv + (size_t) (ss[b] + i) * w + h * hd;
                const int64_t at = h < nh ? 0 : slot(b, h - nh, p);
                if (slot(b, 0, p) < 0) continue;
                const uint16_t * y = h < nh ? q + ((size_t) (ss[b] + i) * nh + h) * hd : kc + at;
                for (int d = 0; d < hd; d++) {
                    double e = x[d];
                    if (d < half) e = (double) x[d] * cs[p * half + d] - (double) x[d + half] * sn[p * half + d];
                    else if (d < rot) e = (double) x[d] * cs[p * half + d - half] + (double) x[d - half] * sn[p * half + d - half];
                    if (std::isnan(e) ? !std::isnan(dec(y[d])) : !(std::fabs(dec(y[d]) - e) <= std::fabs(e) * (g_bf ? 0.0040 : 0.0005) + 1e-6)) {
                        std::fprintf(stderr, "append: row %d head %d dim %d: %g, not %g\n", i, h, d, dec(y[d]), e);
                        return 1;
                    }
                }
            }
    const size_t wsb = gsvk_attn_paged_workspace_bytes(&kv, tokens, nh, max_new, max_keys, window);
    void * ws = wsb ? std::malloc(wsb) : nullptr;
    if (ws) std::memset(ws, 0xff, wsb);
    char * out = (char *) std::malloc((size_t) tokens * nh * hd * (f32 ? 4 : 2));
    std::memset(out, 0x11, (size_t) tokens * nh * hd * (f32 ? 4 : 2));
    float * lse = buf<float>((size_t) tokens * nh);
    for (int i = 0; i < tokens * nh; i++) lse[i] = 77.0f;
    const float scale = 1.0f / std::sqrt((float) hd);
    if (gsvk_op_attn_paged(&kv, q, tokens, nh, (int64_t) nh * hd, max_new, max_keys, scale, window, prefix ? pre : nullptr, out,
                           f32 ? GSVK_TYPE_F32 : kv.type, (int64_t) nh * hd, lse, ws, wsb, nullptr)) {
        std::fprintf(stderr, "%s\n", gsvk::get_error());
        return 1;
    }
    if (poison == 3) {
        std::printf("no access outside the buffers, workspace %zu\n", wsb);
        return 0;
    }
    const auto got = [&](int64_t i) { return f32 ? (double) ((float *) out)[i] : dec(((uint16_t *) out)[i]); };
    double worst = 0, worst_l = 0;
    for (int b = 0; b < B; b++)
        for (int i = 0; i < n[b]; i++)
            for (int h = 0; h < nh; h++) {
                const int p = tot[b] - n[b] + i, row = ss[b] + i;
                const int hi = std::min(tot[b], std::max(p + 1, prefix)), lo = window ? std::max(0, p - window + 1) : 0;
                std::vector<double> sc;
                std::vector<int> key;
                double m = -INFINITY, z = 0;
                for (int j = lo; j < hi; j++) {
                    const int64_t at = slot(b, h / G, j);
                    if (at < 0) continue;
                    double s = 0;
                    for (int d = 0; d < hd; d++) s += dec(q[((size_t) row * nh + h) * hd + d]) * dec(kc[at + d]);
                    sc.push_back(s * scale);
                    key.push_back(j);
                    m = std::max(m, s * scale);
                }
                for (double & s : sc) z += s = std::exp(s - m);
                const double l = sc.empty() ? -INFINITY : m + std::log(z);
                if (std::isnan(z)) {
                    if (!std::isnan(got(((int64_t) row * nh + h) * hd))) return 1;
                    continue;
                }
                if (std::isinf(l) ? lse[row * nh + h] != l : !(std::fabs(lse[row * nh + h] - l) < 1e-4)) {
                    std::fprintf(stderr, "lse: seq %d row %d head %d: %g, not %g\n", b, i, h, lse[row * nh + h], l);
                    return 1;
                }
                for (int d = 0; d < hd; d++) {
                    double y = 0, mag = 0;
                    for (size_t e = 0; e < sc.size(); e++) {
                        const double v = dec(vc[slot(b, h / G, key[e]) + d]);
                        y += sc[e] / z * v;
                        mag += sc[e] / z * std::fabs(v);
                    }
                    const double off = std::fabs(got(((int64_t) row * nh + h) * hd + d) - y) / (mag + 1e-9);
                    if (!(off <= (g_bf ? 0.0085 : 0.0011))) {
                        std::fprintf(stderr, "seq %d row %d head %d dim %d: %g, not %g\n", b, i, h, d, got(((int64_t) row * nh + h) * hd + d), y);
                        return 1;
                    }
                    worst = std::max(worst, off);
                }
                worst_l = 0;
            }
    for (int i = T * nh; i < tokens * nh; i++)
        if (lse[i] != 77.0f) return 1;
    std::printf("hd %d nh %d nkv %d: %d rows, off by %.1e of the values' sizes, workspace %zu\n", hd, nh, nkv, T, worst, wsb);
    return 0;
}
