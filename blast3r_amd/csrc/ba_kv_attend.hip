// Attention over the 8-bit key/value cache.
//
// For a row of queries q and the keys j that it sees,  o = sum_j p_j v_j / sum_j p_j,  p_j = exp(c q.k_j - m):
// one pass over the cache with a running reference m, so that the scores never leave the registers.
//
// A wave takes a tile of query rows (rows that share a cache head: the tokens of a sequence times the query
// heads of that cache head) and walks over blocks of 64 tokens.  The block's bytes go from memory to
// registers in the layout that the matrix instructions want, without LDS:
//   scores   S^T = K Q^T: lane (n, g) of COLS x NG holds, of every key block b, 8-element pieces of a key row;
//            which token a key row of the product stands for is free, and is chosen so that
//   products O^T = V^T P^T: the lane's results S are those of 64 / NG consecutive tokens for query column n,
//            which is the layout of the second operand (P) as it stands, and the values, kept as (dim, 64),
//            are read as consecutive bytes of a row.
// COLS = 16 (16 x 16 x 32 products) is for at most 16 rows, COLS = 32 (32 x 32 x 16) for more, with NCB tiles
// of 32 rows to a wave.  Codes become fp16, which holds each of them exactly; queries are scaled by a power of
// two of their row to fp16, exactly for bf16 and fp16 queries up to 2^-28 of the row's largest element; sums
// are fp32.
//
// Factors: a block's key factor goes into the constant c, its value factor into the exponent: with z = c q.k
// and lv = log2(value factor), m follows z + lv, so that the weights exp2(z + lv - m) that meet the codes of
// the values are at most 2^14 whatever the factors are, and the denominator adds their sums divided by the
// value factor.  The weights of a block whose values are small beside others' may vanish in fp16 and still
// make up the denominator, so that is summed in fp32 before the weights are rounded to fp16 (11 bits, at the
// precision of the outputs or beyond).  m is moved only when a score passes it by 2^8; until then the products
// need no rescaling.
//
// The waves of a workgroup share rows and split the blocks (few rows; joined through LDS), or share the
// blocks and split the rows.  With few rows in all the blocks of a sequence are further cut into n_splits
// parts, whose sums k_kv_join adds in order.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ba_common.h"
#include "ba_error.h"
#include "ba_hip.h"
#include "ba_token.h"

namespace ba {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16 __attribute__((ext_vector_type(16)));

#define AT_T 256
#define AT_WAVES 4
#define AT_MIN_BLOCKS 4      // a split part has at least so many blocks: one for each wave

template <int COLS> struct Mma;
template <> struct Mma<16> {
    typedef f4 acc;
    static __device__ __forceinline__ acc run(h8 a, h8 b, acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    // token of the block that row m of key block b stands for
    static __device__ __forceinline__ int token(int b, int m) { return 16 * (m >> 2) + 4 * b + (m & 3); }
    // element of a 16-row tile that accumulator r of lane group g holds
    static __device__ __forceinline__ int row(int g, int r) { return 4 * g + r; }
};
template <> struct Mma<32> {
    typedef f16 acc;
    static __device__ __forceinline__ acc run(h8 a, h8 b, acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ int token(int b, int m) { return 32 * ((m >> 2) & 1) + 16 * b + 4 * (m >> 3) + (m & 3); }
    static __device__ __forceinline__ int row(int g, int r) { return 8 * (r >> 2) + 4 * g + (r & 3); }
};

// 8 codes to fp16
template <int KT>
__device__ __forceinline__ h8 codes8(uint2 w) {
    h8 r;
    auto put = [&](int i, h2 x) { r[2 * i] = x[0]; r[2 * i + 1] = x[1]; };
    if constexpr (KT == BA_FP8) {
        put(0, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w.x, 1.0f, false));
        put(1, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w.x, 1.0f, true));
        put(2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w.y, 1.0f, false));
        put(3, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w.y, 1.0f, true));
    } else {
        // fp16 with the bits 0x6400 + u is 1024 + u: the code plus 128 there, less 1152
        const uint32_t a = w.x ^ 0x80808080u, b = w.y ^ 0x80808080u;
        const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
        put(0, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) - off);
        put(1, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) - off);
        put(2, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) - off);
        put(3, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) - off);
    }
    return r;
}

// What a sequence of the call has: its rows and its length.
struct AtSeq {
    int64_t row0;
    int n, len;
    int rows;                // of its n rows, those within max_rows
};

__device__ __forceinline__ AtSeq at_seq(const ba_kv_attend_args& a, int s) {
    int64_t row0 = (int64_t)s * a.rows_per_seq, n = a.rows_per_seq;
    if (a.offsets) {
        row0 = a.offsets[s];
        n = (int64_t)a.offsets[s + 1] - row0;
    }
    if (row0 < 0 || row0 > a.n_rows || n < 0) { row0 = 0; n = 0; }
    n = n < a.n_rows - row0 ? n : a.n_rows - row0;
    int64_t len = a.lengths[s];
    const int64_t most = (int64_t)a.n_pages * 64;
    len = len < 0 ? 0 : len < most ? len : most;
    return {row0, (int)n, (int)len, (int)(n < a.max_rows ? n : a.max_rows)};
}

// Blocks [lo, hi) that rows [row, row + rows) (of n * group rows) see, and of these the ones of part sp.
__device__ __forceinline__ void at_blocks(const ba_kv_attend_args& a, const AtSeq& q, int group, int64_t row, int rows, int sp,
                                          int& lo, int& hi) {
    const int64_t all = (int64_t)q.rows * group, last = row + rows < all ? row + rows : all;
    if (row >= last) { lo = hi = 0; return; }
    const int64_t p0 = (int64_t)q.len - q.n + row / group, p1 = (int64_t)q.len - q.n + (last - 1) / group;
    const int64_t keys = a.causal ? p1 + 1 : (int64_t)q.len;
    int64_t first = a.window > 0 ? p0 - a.window + 1 : 0;
    if (first < 0) first = 0;
    if (keys <= first) { lo = hi = 0; return; }
    const int b0 = (int)(first / 64), b1 = (int)((keys + 63) / 64);
    int per = (b1 - b0 + a.n_splits - 1) / a.n_splits;
    per = per < AT_MIN_BLOCKS ? AT_MIN_BLOCKS : per;
    lo = b0 + sp * per < b1 ? b0 + sp * per : b1;
    hi = lo + per < b1 ? lo + per : b1;
}

// rows of a workgroup's tile
template <int COLS, int NCB, int WR> constexpr int tile_rows() { return COLS * NCB * WR; }

// partial sums of a row and part: dim floats, and the reference and the denominator
__device__ __forceinline__ float* part_sum(const ba_kv_attend_args& a, int64_t row, int head, int sp) {
    return (float*)a.workspace + ((row * a.q_heads + head) * a.n_splits + sp) * (int64_t)a.dim;
}
__device__ __forceinline__ float2* part_ref(const ba_kv_attend_args& a, int64_t row, int head, int sp) {
    return (float2*)((float*)a.workspace + a.n_rows * a.q_heads * a.n_splits * (int64_t)a.dim) + (row * a.q_heads + head) * a.n_splits + sp;
}

__device__ __forceinline__ void store_out4(const ba_kv_attend_args& a, int64_t row, int head, int d, f4 v, bool wide) {
    const int64_t at = row * a.o_st + head * a.o_sh + d;
    const float x[4] = {v[0], v[1], v[2], v[3]};
    if (a.dtype == BA_F16) {
        _Float16* o = (_Float16*)a.o + at;
        if (wide) store_vec<_Float16, 4>(o, x);
        else for (int i = 0; i < 4; ++i) o[i] = (_Float16)x[i];
    } else {
        __bf16* o = (__bf16*)a.o + at;
        if (wide) store_vec<__bf16, 4>(o, x);
        else for (int i = 0; i < 4; ++i) o[i] = (__bf16)x[i];
    }
}

#define AT_NONE -1.0e30f      // reference of a row that has seen no key
#define AT_MOVE 8.0f          // m is moved when a score passes it by so much (log2)
#define AT_LIFT 6.0f          // weights at m are 2^6: with AT_MOVE at most 2^14, and fp16 is normal down to 2^-20 of m

// WR waves split the rows of the workgroup's tile, 4 / WR the blocks.
template <int D, int KT, int COLS, int NCB, int WR>
__global__ void __launch_bounds__(AT_T, COLS == 16 && D <= 128 ? 3 : 1) k_kv_attend(ba_kv_attend_args a, int n_tiles, int wide) {
    typedef Mma<COLS> M;
    typedef typename M::acc acc;
    constexpr int NG = 64 / COLS, NB = NG, CREG = COLS * COLS / 64, TPL = 64 / NG;
    constexpr int KS = D / (8 * NG), DB = D / COLS, PS = TPL / 8, WK = AT_WAVES / WR, ROWS = tile_rows<COLS, NCB, WR>();
    __shared__ float2 ref_sh[WK > 1 ? AT_WAVES * COLS * NCB : 1];
    __shared__ f4 sum_sh[WK > 1 ? 2 * COLS * NCB * D / 4 : 1];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave % WR, wk = wave / WR;
    const int n = lane % COLS, g = lane / COLS;
    unsigned id = xcd_block(blockIdx.x, gridDim.x);
    const int tile = (int)(id % (unsigned)n_tiles);
    id /= (unsigned)n_tiles;
    const int sp = (int)(id % (unsigned)a.n_splits);
    id /= (unsigned)a.n_splits;
    const int kh = (int)(id % (unsigned)a.heads), s = (int)(id / (unsigned)a.heads);
    const int group = a.q_heads / a.heads;
    const AtSeq q = at_seq(a, s);
    const int64_t all = (int64_t)q.rows * group, tile0 = (int64_t)tile * ROWS;
    if (tile0 >= all) return;
    int lo, hi;
    at_blocks(a, q, group, tile0, ROWS, sp, lo, hi);
    if (lo >= hi && a.n_splits > 1) return;                  // k_kv_join knows which parts there are

    // queries: row, its position, its elements as fp16 and the power of two that they were divided by
    const int64_t row0 = tile0 + wr * COLS * NCB;
    if constexpr (WK == 1)
        if (row0 >= all) return;
    h8 qf[NCB][KS];
    float qc[NCB];
    int64_t pos[NCB];
#pragma unroll
    for (int c = 0; c < NCB; ++c) {
        const int64_t r = row0 + c * COLS + n, rc = r < all ? r : all - 1;
        const int64_t i = rc / group;
        const int head = kh * group + (int)(rc - i * group);
        pos[c] = (int64_t)q.len - q.n + i;
        float x[KS][8];
        uint32_t top = 0;
        const int64_t at = (q.row0 + i) * a.q_st + head * a.q_sh + g * (D / NG);
#pragma unroll
        for (int t = 0; t < KS; ++t) {
            if (a.dtype == BA_F16) {
                const _Float16* p = (const _Float16*)a.q + at + 8 * t;
                if (wide) load_vec<_Float16, 8>(p, x[t]);
                else for (int j = 0; j < 8; ++j) x[t][j] = (float)p[j];
            } else {
                const __bf16* p = (const __bf16*)a.q + at + 8 * t;
                if (wide) load_vec<__bf16, 8>(p, x[t]);
                else for (int j = 0; j < 8; ++j) x[t][j] = (float)p[j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, __builtin_bit_cast(uint32_t, x[t][j]) & 0x7fffffffu);
        }
#pragma unroll
        for (int m = COLS; m < 64; m <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m));
        int e = (int)(top >> 23) - 127;                      // the row's largest element is in [2^e, 2^(e+1))
        e = e < -100 ? -100 : e > 127 ? 127 : e;
        const float up = __builtin_bit_cast(float, (uint32_t)(14 - e + 127) << 23);
        qc[c] = a.scale * 1.44269504088896341f * __builtin_bit_cast(float, (uint32_t)(e - 14 + 127) << 23);
#pragma unroll
        for (int t = 0; t < KS; ++t)
#pragma unroll
            for (int j = 0; j < 8; ++j) qf[c][t][j] = (_Float16)(x[t][j] * up);
    }
    // positions of the wave's rows, for the choice between blocks that all rows see whole and others
    const int64_t last = row0 + COLS * NCB < all ? row0 + COLS * NCB : all;
    const int64_t pmin = (int64_t)q.len - q.n + row0 / group, pmax = (int64_t)q.len - q.n + (last - 1) / group;
    const int64_t whole_hi = a.causal ? pmin + 1 : (int64_t)q.len;                 // tokens below it are seen by all rows
    const int64_t whole_lo = a.window > 0 ? pmax - a.window + 1 : 0;               // from it on too

    if constexpr (WR > 1) {                                  // the blocks that this wave's rows see
        if (a.causal && (int64_t)hi * 64 > pmax + 64) hi = pmax < 0 ? lo : (int)(pmax / 64) + 1;
        const int64_t first = a.window > 0 ? pmin - a.window + 1 : 0;
        if (first / 64 > lo) lo = (int)(first / 64 < hi ? first / 64 : hi);
    }

    acc o[NCB][DB];
    float m[NCB], l[NCB];
#pragma unroll
    for (int c = 0; c < NCB; ++c) {
        m[c] = AT_NONE;
        l[c] = 0.0f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < CREG; ++r) o[c][d][r] = 0.0f;
    }

    const int32_t* pages = a.pages + (int64_t)s * a.pages_stride;
    const uint8_t* kb = (const uint8_t*)a.k + (int64_t)kh * 64 * D;
    const uint8_t* vb = (const uint8_t*)a.v + (int64_t)kh * 64 * D;
    const int64_t step = (int64_t)a.heads * 64 * D;
    uint2 kr[NB][KS], vr[DB][PS];
    auto load_keys = [&](int64_t page) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint8_t* p = kb + page * step + M::token(b, n) * D + g * (D / NG);
            if constexpr (KS % 2 == 0) {
#pragma unroll
                for (int t = 0; t < KS; t += 2) {
                    const uint4 w = *(const uint4*)(p + 8 * t);
                    kr[b][t] = make_uint2(w.x, w.y);
                    kr[b][t + 1] = make_uint2(w.z, w.w);
                }
            } else {
#pragma unroll
                for (int t = 0; t < KS; ++t) kr[b][t] = *(const uint2*)(p + 8 * t);
            }
        }
    };
    auto load_values = [&](int64_t page) {
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            const uint8_t* p = vb + page * step + (d * COLS + n) * 64 + g * TPL;
#pragma unroll
            for (int t = 0; t < PS; t += 2) {
                const uint4 w = *(const uint4*)(p + 8 * t);
                vr[d][t] = make_uint2(w.x, w.y);
                vr[d][t + 1] = make_uint2(w.z, w.w);
            }
        }
    };
    auto page_of = [&](int b) -> int64_t {
        const int64_t p = b < hi ? pages[b] : -1;
        return p < a.n_blocks ? p : -1;
    };

    int blk = lo + wk;
    int64_t page = page_of(blk);
    if (page >= 0) { load_keys(page); load_values(page); }
    while (blk < hi) {
        const int64_t next = page_of(blk + WK);
        if (page >= 0) {
            const float2 f = *(const float2*)(a.scales + (page * a.heads + kh) * 2);
            acc sc[NCB][NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int c = 0; c < NCB; ++c)
#pragma unroll
                    for (int r = 0; r < CREG; ++r) sc[c][b][r] = 0.0f;
#pragma unroll
                for (int t = 0; t < KS; ++t) {
                    const h8 kf = codes8<KT>(kr[b][t]);
#pragma unroll
                    for (int c = 0; c < NCB; ++c) sc[c][b] = M::run(kf, qf[c][t], sc[c][b]);
                }
            }
            if (next >= 0) load_keys(next);
            const float lv = __builtin_amdgcn_logf(f.y), iv = 1.0f / f.y;
            const int64_t t0 = (int64_t)blk * 64;
            const bool masked = t0 + 64 > whole_hi || t0 < whole_lo;
            if (t0 + 64 > q.len) {                           // tokens that were never written: their codes may be anything
                const int over = q.len - (int)t0 - g * TPL;  // the lane's tokens from here on
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int t = 0; t < PS; ++t) {
                        const int x = over - 8 * t, y = x - 4;
                        vr[d][t].x &= x >= 4 ? ~0u : x <= 0 ? 0u : (1u << (8 * x)) - 1u;
                        vr[d][t].y &= y >= 4 ? ~0u : y <= 0 ? 0u : (1u << (8 * y)) - 1u;
                    }
            }
            h8 pf[NCB][PS];
#pragma unroll
            for (int c = 0; c < NCB; ++c) {
                const float cz = f.x * qc[c];
                int seen_lo = 0, seen_hi = TPL - 1;          // the lane's tokens that the row sees
                if (masked) {
                    const int64_t base = t0 + g * TPL;
                    const int64_t e = (a.causal && pos[c] < q.len ? pos[c] : (int64_t)q.len - 1) - base;
                    const int64_t b = a.window > 0 ? pos[c] - a.window + 1 - base : -1;
                    seen_hi = (int)(e < -1 ? -1 : e > TPL - 1 ? TPL - 1 : e);
                    seen_lo = (int)(b < 0 ? 0 : b > TPL ? TPL : b);
#pragma unroll
                    for (int b2 = 0; b2 < NB; ++b2)
#pragma unroll
                        for (int r = 0; r < CREG; ++r) {
                            const int t = b2 * CREG + r;
                            sc[c][b2][r] = t >= seen_lo && t <= seen_hi ? sc[c][b2][r] : -3.0e38f;
                        }
                }
                float top = sc[c][0][0];
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < CREG; ++r) top = fmaxf(top, sc[c][b][r]);
                top = seen_lo <= seen_hi ? fmaf(top, cz, lv) : AT_NONE;         // a block without a seen token moves nothing
                if (__any(top > m[c] + AT_MOVE)) {
                    float now = fmaxf(top, m[c]);
#pragma unroll
                    for (int k = COLS; k < 64; k <<= 1) now = fmaxf(now, __shfl_xor(now, k));
                    const float by = __builtin_amdgcn_exp2f(m[c] - now);
                    m[c] = now;
                    l[c] *= by;
#pragma unroll
                    for (int d = 0; d < DB; ++d)
#pragma unroll
                        for (int r = 0; r < CREG; ++r) o[c][d][r] *= by;
                }
                const float off = lv - m[c] + AT_LIFT;
                float sum = 0.0f;
#pragma unroll
                for (int t = 0; t < PS; ++t)
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const int k = 8 * t + j;
                        float x = __builtin_amdgcn_exp2f(fmaf(sc[c][k / CREG][k % CREG], cz, off));
                        float y = __builtin_amdgcn_exp2f(fmaf(sc[c][(k + 1) / CREG][(k + 1) % CREG], cz, off));
                        if (masked) {
                            x = k >= seen_lo && k <= seen_hi ? x : 0.0f;
                            y = k + 1 >= seen_lo && k + 1 <= seen_hi ? y : 0.0f;
                        }
                        const h2 p = {(_Float16)x, (_Float16)y};
                        sum += x + y;                        // before rounding: see the factors above
                        pf[c][t][j] = p[0];
                        pf[c][t][j + 1] = p[1];
                    }
                l[c] = fmaf(sum, iv, l[c]);
            }
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int t = 0; t < PS; ++t) {
                    const h8 vf = codes8<KT>(vr[d][t]);
#pragma unroll
                    for (int c = 0; c < NCB; ++c) o[c][d] = M::run(vf, pf[c][t], o[c][d]);
                }
            if (next >= 0) load_values(next);
        } else if (next >= 0) {
            load_keys(next);
            load_values(next);
        }
        page = next;
        blk += WK;
    }
#pragma unroll
    for (int c = 0; c < NCB; ++c)
#pragma unroll
        for (int k = COLS; k < 64; k <<= 1) l[c] += __shfl_xor(l[c], k);

    if constexpr (WK > 1) {                                  // one reference for the waves, then their sums in order
        if (g == 0)
#pragma unroll
            for (int c = 0; c < NCB; ++c) ref_sh[wave * COLS * NCB + c * COLS + n] = make_float2(m[c], l[c]);
        __syncthreads();
#pragma unroll
        for (int c = 0; c < NCB; ++c) {
            float2 r[AT_WAVES];
            float top = AT_NONE;
#pragma unroll
            for (int w = 0; w < AT_WAVES; ++w) {
                r[w] = ref_sh[w * COLS * NCB + c * COLS + n];
                top = fmaxf(top, r[w].x);
            }
            const float by = __builtin_amdgcn_exp2f(m[c] - top);
            m[c] = top;
            l[c] = 0.0f;
#pragma unroll
            for (int w = 0; w < AT_WAVES; ++w) l[c] = fmaf(r[w].y, __builtin_amdgcn_exp2f(r[w].x - top), l[c]);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int k = 0; k < CREG; ++k) o[c][d][k] *= by;
        }
        auto at = [&](int buf, int c, int d, int r4) { return ((buf * NCB + c) * DB + d) * (CREG / 4) * 64 + r4 * 64 + lane; };
        auto put = [&](int buf) {
#pragma unroll
            for (int c = 0; c < NCB; ++c)
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int r = 0; r < CREG; r += 4)
                        sum_sh[at(buf, c, d, r / 4)] = (f4){o[c][d][r], o[c][d][r + 1], o[c][d][r + 2], o[c][d][r + 3]};
        };
        auto add = [&](int buf) {
#pragma unroll
            for (int c = 0; c < NCB; ++c)
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int r = 0; r < CREG; r += 4) {
                        const f4 x = sum_sh[at(buf, c, d, r / 4)];
#pragma unroll
                        for (int k = 0; k < 4; ++k) o[c][d][r + k] += x[k];
                    }
        };
        if (wk >= 2) put(wk - 2);
        __syncthreads();
        if (wk < 2) add(wk);
        __syncthreads();
        if (wk == 1) put(0);
        __syncthreads();
        if (wk != 0) return;
        add(0);
    }

#pragma unroll
    for (int c = 0; c < NCB; ++c) {
        const int64_t r = row0 + c * COLS + n;
        if (r >= all) continue;
        const int64_t i = r / group, row = q.row0 + i;
        const int head = kh * group + (int)(r - i * group);
        if (a.n_splits > 1) {
            float* w = part_sum(a, row, head, sp);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int k = 0; k < CREG; k += 4)
                    *(f4*)(w + d * COLS + M::row(g, k)) = (f4){o[c][d][k], o[c][d][k + 1], o[c][d][k + 2], o[c][d][k + 3]};
            if (g == 0) *part_ref(a, row, head, sp) = make_float2(m[c], l[c]);
            continue;
        }
        // !(l == 0): a row without keys has l = 0, a NaN among its keys or queries has to come through
        const float inv = l[c] == 0.0f ? 0.0f : 1.0f / l[c];
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int k = 0; k < CREG; k += 4)
                store_out4(a, row, head, d * COLS + M::row(g, k),
                           (f4){o[c][d][k] * inv, o[c][d][k + 1] * inv, o[c][d][k + 2] * inv, o[c][d][k + 3] * inv}, wide != 0);
        if (a.lse && g == 0)
            a.lse[row * a.q_heads + head] = l[c] == 0.0f ? -__builtin_inff() : 0.693147180559945309f * (m[c] - AT_LIFT + __builtin_amdgcn_logf(l[c]));
    }
}

// The parts of each row joined: a thread takes 4 elements, `lanes` groups of threads the parts in turn.
__global__ void __launch_bounds__(AT_T) k_kv_join(ba_kv_attend_args a, int tile_rows, int lanes, int wide) {
    __shared__ f4 sum_sh[AT_T];
    __shared__ float den_sh[AT_T];
    const int quads = a.dim / 4, unit = threadIdx.x / quads, d = threadIdx.x % quads * 4;
    const int per_wg = AT_T / quads / lanes;                 // rows of a workgroup
    const int64_t rh = (int64_t)blockIdx.x * per_wg + unit / lanes;
    const int lane = unit % lanes;
    const int64_t row = rh / a.q_heads;
    const int head = (int)(rh - row * a.q_heads);
    const bool mine = unit / lanes < per_wg && row < a.n_rows;
    f4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    float den = 0.0f, top = AT_NONE;
    bool covered = false;
    if (mine) {
        int s = 0;                                           // the row's sequence
        if (a.offsets) {
            int e = a.n_seqs;                                // the last s with offsets[s] <= row
            while (e - s > 1) {
                const int c = (s + e) >> 1;
                if (a.offsets[c] <= row) s = c; else e = c;
            }
        } else {
            s = (int)(row / a.rows_per_seq);
        }
        AtSeq q = {0, 0, 0, 0};
        if (s < a.n_seqs) q = at_seq(a, s);
        const int64_t i = row - q.row0;
        const int group = a.q_heads / a.heads;
        covered = i >= 0 && i < q.rows;
        if (covered) {
            const int64_t r = i * group + head % group, tile0 = r / tile_rows * tile_rows;
            int n = 0, lo, hi;
            for (; n < a.n_splits; ++n) {
                at_blocks(a, q, group, tile0, tile_rows, n, lo, hi);
                if (lo >= hi) break;
            }
            for (int p = 0; p < n; ++p) top = fmaxf(top, part_ref(a, row, head, p)->x);
            for (int p = lane; p < n; p += lanes) {
                const float2 f = *part_ref(a, row, head, p);
                const float by = __builtin_amdgcn_exp2f(f.x - top);
                const f4 x = *(const f4*)(part_sum(a, row, head, p) + d);
                den = fmaf(f.y, by, den);
#pragma unroll
                for (int k = 0; k < 4; ++k) sum[k] = fmaf(x[k], by, sum[k]);
            }
        }
    }
    sum_sh[threadIdx.x] = sum;
    den_sh[threadIdx.x] = den;
    __syncthreads();
    if (!covered || lane != 0) return;
    for (int k = 1; k < lanes; ++k) {
        sum += sum_sh[threadIdx.x + k * quads];
        den += den_sh[threadIdx.x + k * quads];
    }
    const float inv = den == 0.0f ? 0.0f : 1.0f / den;
    store_out4(a, row, head, d, sum * inv, wide != 0);
    if (a.lse && d == 0)
        a.lse[row * a.q_heads + head] = den == 0.0f ? -__builtin_inff() : 0.693147180559945309f * (top - AT_LIFT + __builtin_amdgcn_logf(den));
}

// The variant for a call: at most 16 rows of a cache head go through 16 columns, more through 32 (one or two
// tiles of them to a wave), and from 65 rows on the waves split the rows.
struct AtShape { int cols, ncb, wr; };
static AtShape at_shape(int64_t rows, int dim) {
    if (rows <= 16) return {16, 1, 1};
    if (rows <= 32) return {32, 1, 1};
    if (rows <= 128 || dim > 128) return {32, 1, 4};
    return {32, 2, 4};
}

template <int D, int KT>
static int launch_attend(const ba_kv_attend_args& a, AtShape v, unsigned nb, int tiles, int wide, hipStream_t st) {
    if (v.cols == 16) hipLaunchKernelGGL((k_kv_attend<D, KT, 16, 1, 1>), dim3(nb), dim3(AT_T), 0, st, a, tiles, wide);
    else if (v.wr == 1) hipLaunchKernelGGL((k_kv_attend<D, KT, 32, 1, 1>), dim3(nb), dim3(AT_T), 0, st, a, tiles, wide);
    else if (v.ncb == 1) hipLaunchKernelGGL((k_kv_attend<D, KT, 32, 1, 4>), dim3(nb), dim3(AT_T), 0, st, a, tiles, wide);
    else if constexpr (D <= 128) hipLaunchKernelGGL((k_kv_attend<D, KT, 32, 2, 4>), dim3(nb), dim3(AT_T), 0, st, a, tiles, wide);
    BA_LAUNCHED();
    return BA_OK;
}

}  // namespace ba

using namespace ba;

extern "C" int32_t ba_kv_attend_splits(int32_t n_seqs, int32_t heads, int32_t q_heads, int32_t dim, int64_t max_rows,
                                       int32_t n_pages) {
    if (n_seqs < 1 || heads < 1 || q_heads < heads || max_rows < 1 || n_pages < 1) return 1;
    const int64_t rows = max_rows * (q_heads / heads);
    const AtShape v = at_shape(rows, dim);
    const int64_t tile = v.cols * v.ncb * v.wr, base = (int64_t)n_seqs * heads * ((rows + tile - 1) / tile);
    const int64_t most = (n_pages + AT_MIN_BLOCKS - 1) / AT_MIN_BLOCKS;
    int64_t n = (1024 + base - 1) / base;                    // four workgroups for each of 256 CUs
    n = n < most ? n : most;
    return (int32_t)(n < 1 ? 1 : n);
}

extern "C" int64_t ba_kv_attend_workspace_bytes(int64_t n_rows, int32_t q_heads, int32_t dim, int32_t n_splits) {
    return n_splits > 1 && n_rows > 0 ? n_rows * q_heads * n_splits * ((int64_t)dim + 2) * 4 : 0;
}

extern "C" int ba_kv_attend(const ba_kv_attend_args* args, void* stream) {
    clear_error();
    BA_REQUIRE(args != nullptr, "null args");
    const ba_kv_attend_args& a = *args;
    BA_REQUIRE(a.n_blocks >= 0 && a.heads >= 1 && a.heads <= 65536 && a.n_seqs >= 0 && a.n_pages >= 0, "attention: bad sizes");
    BA_REQUIRE(a.dim == 32 || a.dim == 64 || a.dim == 96 || a.dim == 128 || a.dim == 256,
               "attention: head size must be 32, 64, 96, 128 or 256");
    BA_REQUIRE(a.q_heads >= 1 && a.q_heads <= 65536 && a.q_heads % a.heads == 0, "attention: query heads must be a multiple of the cache's");
    BA_REQUIRE(a.bits == BA_FP8 || a.bits == BA_INT8, "attention: bits must be 0 (e4m3) or 1 (int8)");
    BA_REQUIRE(a.dtype == BA_F16 || a.dtype == BA_BF16, "attention: queries must be fp16 or bf16");
    BA_REQUIRE(a.n_rows >= 0 && a.rows_per_seq >= 0 && a.max_rows >= 0 && a.window >= 0 && a.n_rows < (int64_t)1 << 31 &&
                   a.max_rows < (int64_t)1 << 31 && a.n_pages < 1 << 24, "attention: bad sizes");
    BA_REQUIRE(a.scale > 0.0f && a.scale < 1.0e30f, "attention: scale must be positive");
    BA_REQUIRE(a.n_splits >= 1 && a.n_splits <= 65536, "attention: n_splits must be in [1, 65536]");
    if (a.n_rows == 0 || a.n_seqs == 0 || a.max_rows == 0) return BA_OK;
    BA_REQUIRE(a.offsets != nullptr || a.rows_per_seq >= 1, "attention: rows without sequences");
    BA_REQUIRE(a.q && a.o && a.lengths, "null pointer");
    BA_REQUIRE((a.n_pages == 0 || a.pages) && (a.n_blocks == 0 || (a.k && a.v && a.scales)), "null pointer");
    BA_REQUIRE((uintptr_t)a.k % 16 == 0 && (uintptr_t)a.v % 16 == 0 && (uintptr_t)a.scales % 8 == 0,
               "attention: k and v must be aligned to 16 bytes, scales to 8");
    const int group = a.q_heads / a.heads;
    const int64_t rows = a.max_rows * group;
    const AtShape v = at_shape(rows, a.dim);
    const int tile = v.cols * v.ncb * v.wr;
    const int64_t tiles = (rows + tile - 1) / tile;
    // a launch has less than 2^32 threads
    BA_REQUIRE(tiles <= ((int64_t)1 << 23) / a.n_seqs / a.heads / a.n_splits, "attention: too many tiles for a call (max_rows is the bound that counts)");
    if (a.n_splits > 1) {
        BA_REQUIRE(a.workspace && (uintptr_t)a.workspace % 16 == 0, "null pointer");
        BA_REQUIRE(a.workspace_bytes >= ba_kv_attend_workspace_bytes(a.n_rows, a.q_heads, a.dim, a.n_splits), "attention: workspace too small");
    }
    const unsigned nb = (unsigned)(tiles * a.n_seqs * a.heads * a.n_splits);
    // loads of 8 queries, stores of 4 outputs
    const int wide = (uintptr_t)a.q % 16 == 0 && (uintptr_t)a.o % 8 == 0 && a.q_st % 8 == 0 && a.q_sh % 8 == 0 && a.o_st % 4 == 0 && a.o_sh % 4 == 0;
    hipStream_t st = (hipStream_t)stream;
    int rc = BA_ERR_UNSUPPORTED;
#define BA_AT_D(D) \
    case D: rc = a.bits == BA_FP8 ? launch_attend<D, BA_FP8>(a, v, nb, (int)tiles, wide, st) : launch_attend<D, BA_INT8>(a, v, nb, (int)tiles, wide, st); break;
    switch (a.dim) { BA_AT_D(32) BA_AT_D(64) BA_AT_D(96) BA_AT_D(128) BA_AT_D(256) }
#undef BA_AT_D
    if (rc != BA_OK || a.n_splits == 1) return rc;
    int lanes = 1;
    while (lanes < a.n_splits && 2 * lanes * (a.dim / 4) <= AT_T) lanes *= 2;
    const int per_wg = AT_T / (a.dim / 4) / lanes;
    const int64_t jobs = a.n_rows * a.q_heads;
    BA_REQUIRE((jobs + per_wg - 1) / per_wg < (int64_t)1 << 24, "attention: too many rows for a call");
    hipLaunchKernelGGL(k_kv_join, dim3((unsigned)((jobs + per_wg - 1) / per_wg)), dim3(AT_T), 0, st, a, tile, lanes, wide);
    BA_LAUNCHED();
    return BA_OK;
}
