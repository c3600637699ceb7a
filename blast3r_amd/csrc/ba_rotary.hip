// Rotary positions: pairs of a head's elements turned by angles that grow with a token's position.
//
// The rotated part of a head (its first `part` elements) is cut into `axes` equal sections, one for
// each coordinate of the position (a sequence has one, an image patch its row and column).  Pair p of
// a section of n elements is (p, p + n/2) in the half layout and (2p, 2p + 1) in the interleaved one:
//   y1 = m (x1 cos t - x2 sin t),  y2 = m (x1 sin t + x2 cos t),  t = position * frequency_p.
// The rest of the head is copied.  The map is m times a rotation, so the gradient of x is the same
// map of the gradient of y with -t (inverse = 1).
//
// Angles: frequency_p is held as turns per position in 64-bit fixed point (2^64 = one turn), so that
// position * turns wraps modulo one turn exactly, at any position; a product in fp32 is off by half a
// radian at position 2^23.  The top bits give the quarter turn and the rest, |t| <= pi/4, whose sine and
// cosine are Taylor sums (remainders below 2e-9).  No table is read or kept.
//
// Bound by memory: 2 bytes in and out of each element against ~25 operations per angle.  A thread makes
// the angles of its pairs once and takes several heads of the token with them (q and k in one launch);
// loads and stores are 16 bytes where strides and addresses allow it.  32768 tokens of 40 heads of 128
// (671 MB): 125 us a direction, 5.4 TB/s, as a copy of the same bytes; it was 189 us with 64-bit products
// of strides for every head.  Non-temporal stores: 118 us there, but 135 against 112 at 65536 tokens of 32
// heads of 64, and the next operator reads what they would push out.  Sections that are no whole vectors go by single
// elements (or pairs): 32768 tokens of 32 heads, half of a head, two axes: 42 us for heads of 32 and 168 for 96, where a
// copy of the same bytes would take 25 and 75.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ba_error.h"
#include "ba_hip.h"
#include "ba_token.h"

// every variant of the kernel rounds alike: fused steps are written as fmaf
#pragma clang fp contract(off)

namespace ba {

#define ROT_T 256
#define ROT_B 2

struct RotGrid {
    unsigned n;              // threads that work
    unsigned units, groups;  // vectors (or vector pairs) of a head row; groups of heads
    unsigned rot_units;      // units that rotate; the others copy
    unsigned per;            // heads of a thread
    int64_t first, batch;    // token and batch of thread 0
};

__device__ __forceinline__ void turn_sincos(uint64_t frac, float& s, float& c) {
    const unsigned top = (unsigned)(frac >> 32);
    const unsigned q = (top + 0x20000000u) >> 30;                       // nearest quarter turn
    const float x = (float)(int)(top - (q << 30)) * 1.46291807926715968e-9f;   // 2 pi / 2^32
    const float z = x * x;
    float sn = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);                  // 1/9!, -1/7!
    sn = fmaf(z, sn, 8.3333333e-3f);
    sn = fmaf(z, sn, -1.6666667e-1f);
    sn = fmaf(x * z, sn, x);
    float cs = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);                  // -1/10!, 1/8!
    cs = fmaf(z, cs, -1.3888889e-3f);
    cs = fmaf(z, cs, 4.1666667e-2f);
    cs = fmaf(z, cs, -0.5f);
    cs = fmaf(z, cs, 1.0f);
    const float a = (q & 1) ? cs : sn, b = (q & 1) ? sn : cs;
    s = (q & 2) ? -a : a;
    c = ((q + 1) & 2) ? -b : b;
}

// V elements of type T per vector: 16 bytes, or one (or one pair) where addresses are not aligned.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(ROT_T) k_rotary(ba_rotary_args a, RotGrid g) {
    constexpr int NP = INTER ? V / 2 : V;                               // pairs of a unit
    const unsigned id = blockIdx.x * ROT_T + threadIdx.x;
    if (id >= g.n) return;
    const unsigned u = id % g.units, rest = id / g.units;
    const unsigned hg = rest % g.groups;
    const int64_t t = g.first + rest / g.groups, b = g.batch + blockIdx.y;
    const bool copy = u >= g.rot_units;
    const int n = a.part / a.axes;                                      // elements of a section
    int e0, p0 = 0, ax = 0;
    if (copy) {
        e0 = a.part + (int)(u - g.rot_units) * V;
    } else if (INTER) {
        e0 = (int)u * V;
        ax = e0 / n;
        p0 = (e0 - ax * n) / 2;
    } else {
        const int per_sec = n / 2 / V;
        ax = (int)u / per_sec;
        p0 = ((int)u - ax * per_sec) * V;
        e0 = ax * n + p0;
    }
    float sn[NP], cs[NP];
    if (!copy) {
        const int64_t at = b * a.pos_sb + t * a.pos_st + ax * a.pos_sa;
        const int64_t pos = a.pos_int64 ? ((const int64_t*)a.positions)[at] : (int64_t)((const int32_t*)a.positions)[at];
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            turn_sincos((uint64_t)pos * a.turns[p0 + i], sn[i], cs[i]);
            sn[i] *= a.inverse ? -a.factor : a.factor;
            cs[i] *= a.factor;
        }
    }
    // ROT_B heads at a time: all their loads are under way before the first is used
    const unsigned heads = (unsigned)(a.heads[0] + a.heads[1]);
    const T* xt[2] = {(const T*)a.x[0] + b * a.x_sb[0] + t * a.x_st[0] + e0, (const T*)a.x[1] + b * a.x_sb[1] + t * a.x_st[1] + e0};
    T* yt[2] = {(T*)a.y[0] + b * a.y_sb[0] + t * a.y_st[0] + e0, (T*)a.y[1] + b * a.y_sb[1] + t * a.y_st[1] + e0};
    for (unsigned k = 0; k < g.per; k += ROT_B) {
        float v0[ROT_B][V], v1[ROT_B][V];
        T* y[ROT_B];
#pragma unroll
        for (unsigned j = 0; j < ROT_B; ++j) {
            const unsigned h = hg + (k + j) * g.groups;
            if (k + j >= g.per || h >= heads) break;
            const bool first = h < (unsigned)a.heads[0];
            const int hh = (int)(first ? h : h - a.heads[0]);        // strides of heads are below 2^31: one multiply-add each
            const T* x = (first ? xt[0] : xt[1]) + (int64_t)hh * (first ? (int)a.x_sh[0] : (int)a.x_sh[1]);
            y[j] = (first ? yt[0] : yt[1]) + (int64_t)hh * (first ? (int)a.y_sh[0] : (int)a.y_sh[1]);
            load_vec<T, V>(x, v0[j]);
            if (!INTER && !copy) load_vec<T, V>(x + n / 2, v1[j]);
        }
#pragma unroll
        for (unsigned j = 0; j < ROT_B; ++j) {
            if (k + j >= g.per || hg + (k + j) * g.groups >= heads) break;
            if (!copy) {
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    float& p = INTER ? v0[j][2 * i] : v0[j][i];
                    float& q = INTER ? v0[j][2 * i + 1] : v1[j][i];
                    const float x = p, z = q;
                    p = fmaf(x, cs[i], -(z * sn[i]));
                    q = fmaf(x, sn[i], z * cs[i]);
                }
                if (!INTER) store_vec<T, V>(y[j] + n / 2, v1[j]);
            }
            store_vec<T, V>(y[j], v0[j]);
        }
    }
}

template <typename T, int V>
static int launch_rotary(const ba_rotary_args& a, hipStream_t st) {
    RotGrid g;
    const int heads = a.heads[0] + a.heads[1];
    g.rot_units = (unsigned)(a.interleaved ? a.part / V : a.part / 2 / V);
    bool same = true;                                                   // in place: the rest of the head stays
    for (int w = 0; w < a.n_x; ++w)
        same = same && a.x[w] == a.y[w] && a.x_sb[w] == a.y_sb[w] && a.x_st[w] == a.y_st[w] && a.x_sh[w] == a.y_sh[w];
    g.units = g.rot_units + (same ? 0u : (unsigned)((a.dim - a.part) / V));
    // several heads share a thread's angles once there are threads enough for the chip without that (6144 tokens, 32
    // heads of 64, by 4 times more threads: 15.2 us against 11.7; one head a thread at 32768 tokens: 268 against 125)
    const int64_t tokens = a.B * a.T;
    g.per = 1;
    while (g.per < 8 && (int)g.per < heads && tokens * g.units * (heads / (2 * (int)g.per)) >= 256 * 512) g.per *= 2;
    g.groups = (unsigned)((heads + (int)g.per - 1) / (int)g.per);
    const int64_t per_token = (int64_t)g.units * g.groups, most = ((int64_t)1 << 31) / per_token;
    for (g.batch = 0; g.batch < a.B; g.batch += 65535)
        for (g.first = 0; g.first < a.T; g.first += most) {             // thread numbers stay in 32 bits
            const int64_t now = a.T - g.first < most ? a.T - g.first : most, nb = a.B - g.batch < 65535 ? a.B - g.batch : 65535;
            g.n = (unsigned)(now * per_token);
            const dim3 grid((g.n + ROT_T - 1) / ROT_T, (unsigned)nb);
            if (a.interleaved) hipLaunchKernelGGL((k_rotary<T, V < 2 ? 2 : V, true>), grid, dim3(ROT_T), 0, st, a, g);
            else hipLaunchKernelGGL((k_rotary<T, V, false>), grid, dim3(ROT_T), 0, st, a, g);
            BA_LAUNCHED();
        }
    return BA_OK;
}

template <typename T>
static int rotary_of(const ba_rotary_args& a, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const int n = a.part / a.axes;
    bool wide = (a.interleaved ? n : n / 2) % V == 0 && a.dim % V == 0 && a.part % V == 0;
    for (int w = 0; w < a.n_x; ++w) {
        const int64_t s[6] = {a.x_sb[w], a.x_st[w], a.x_sh[w], a.y_sb[w], a.y_st[w], a.y_sh[w]};
        for (int i = 0; i < 6; ++i) wide = wide && s[i] % V == 0;
        wide = wide && (uintptr_t)a.x[w] % 16 == 0 && (uintptr_t)a.y[w] % 16 == 0;
    }
    return wide ? launch_rotary<T, V>(a, st) : a.interleaved ? launch_rotary<T, 2>(a, st) : launch_rotary<T, 1>(a, st);
}

}  // namespace ba

using namespace ba;

extern "C" int ba_rotary(const ba_rotary_args* args, void* stream) {
    clear_error();
    BA_REQUIRE(args != nullptr, "null args");
    ba_rotary_args a = *args;
    BA_REQUIRE(a.n_x == 1 || a.n_x == 2, "rotary: one or two tensors");
    BA_REQUIRE(a.B >= 0 && a.T >= 0 && a.heads[0] >= 1 && (a.n_x == 1 || a.heads[1] >= 1), "rotary: bad sizes");
    BA_REQUIRE(a.T == 0 || a.B <= ((int64_t)1 << 40) / a.T, "rotary: bad sizes");
    if (a.n_x == 1) a.heads[1] = 0;
    for (int w = 0; w < a.n_x; ++w)
        BA_REQUIRE(a.x_sh[w] > -((int64_t)1 << 31) && a.x_sh[w] < (int64_t)1 << 31 && a.y_sh[w] > -((int64_t)1 << 31) && a.y_sh[w] < (int64_t)1 << 31,
                   "rotary: strides of heads must be below 2^31");
    if (a.T == 1) {                                                     // single tokens: the batch takes their place
        a.T = a.B;
        a.B = 1;
        a.pos_st = a.pos_sb;
        for (int w = 0; w < 2; ++w) { a.x_st[w] = a.x_sb[w]; a.y_st[w] = a.y_sb[w]; }
    }
    BA_REQUIRE(a.heads[0] <= 65536 && a.heads[1] <= 65536, "rotary: bad sizes");
    BA_REQUIRE(a.dim >= 2 && a.dim <= 65536, "rotary: head size must be in [2, 65536]");
    BA_REQUIRE(a.axes >= 1 && a.part >= 2 && a.part <= a.dim && a.part % (2 * a.axes) == 0,
               "rotary: the rotated part must be at most the head and whole pairs for each axis");
    BA_REQUIRE((a.dim - a.part) % 2 == 0 || !a.interleaved, "rotary: an interleaved head must be even");
    BA_REQUIRE(a.dtype >= 0 && a.dtype <= 2, "rotary: dtype must be fp32, fp16 or bf16");
    if (a.B * a.T == 0) return BA_OK;
    BA_REQUIRE(a.positions && a.turns && a.x[0] && a.y[0] && (a.n_x == 1 || (a.x[1] && a.y[1])), "null pointer");
    hipStream_t st = (hipStream_t)stream;
    if (a.dtype == BA_F32) return rotary_of<float>(a, st);
    if (a.dtype == BA_F16) return rotary_of<_Float16>(a, st);
    return rotary_of<__bf16>(a, st);
}
