// The 8-bit key/value cache: rows written into its blocks, and read back.
//
// A block holds 64 tokens of a head, keys as (64, dim) and values as (dim, 64), with one factor for its
// keys and one for its values: x ~ code * factor.  For e4m3 the factor is a power of two, which costs
// such codes no precision (their step follows their size) and makes the product with the factor exact;
// for int8 it is largest / 127.  Tokens come one at a time as well as by frames, so a block's factor may
// have to grow while it fills: its codes are then rewritten with the new one.
//
// One workgroup takes the keys or the values of one block and head that the call touches, so no other
// one writes there: no atomics.  Values are stored transposed because that is how the product with them
// reads them (ba_kv_attend.hip); they pass through LDS, 4 tokens to a word, with rows of 17 words, so that
// the words that a wave writes lie in different banks.
//
// Bound by memory: es bytes in and one out of each element (writing), the other way round (reading).  12288 tokens of
// 16 heads of 64 (75 MB): written in 18 us, read in 13 to 14 (4.1 and 5.6 TB/s); ragged rows of 8 heads of 128 (120 MB): 24
// and 22 us; 131072 tokens read (805 MB): 160 us, 5.0 TB/s; one token for each of 64 sequences of 8 heads of 128: 6.2 us, 7.6
// where every block's codes are made anew.  Writing is the slower one because a workgroup's stores wait for
// the largest of its loads; 8 workgroups to a CU overlap.  Two workgroups of 128 threads or one of 512 in the place of
// one of 256 were slower (32.9 and 31.2 us against 27.8 for the ragged rows).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ba_error.h"
#include "ba_hip.h"
#include "ba_token.h"

// x * (1 / factor) rounds on its own before it is coded
#pragma clang fp contract(off)

namespace ba {

#define KV_T 256
#define KV_FEW 8            // up to so many tokens go to a values block byte by byte
#define KV_ROW 68           // bytes of a row of the values tile: 64 and one word

// this workgroup's share of the call: rows [row, row + n) are tokens [at, at + n) of block `page`; at < 64
struct KvShare {
    int64_t page, row;
    int at, n;
};

__device__ __forceinline__ bool kv_share(const ba_kv_args& a, int s, int slot_of_call, KvShare& r) {
    int64_t row0 = (int64_t)s * a.rows_per_seq, count = a.rows_per_seq;
    if (a.offsets) {
        row0 = a.offsets[s];
        count = (int64_t)a.offsets[s + 1] - row0;
    }
    const int64_t start = a.starts[s];
    count = count < a.max_rows ? count : a.max_rows;
    if (row0 < 0 || row0 >= a.n_rows || start < 0) return false;
    count = count < a.n_rows - row0 ? count : a.n_rows - row0;
    const int64_t slot = start / 64 + slot_of_call;
    const int64_t lo = slot_of_call ? slot * 64 : start, end = start + count, hi = end < slot * 64 + 64 ? end : slot * 64 + 64;
    if (lo >= hi || slot >= a.n_pages) return false;
    r.page = a.pages[(int64_t)s * a.pages_stride + slot];
    r.row = row0 + lo - start;
    r.at = (int)(lo - slot * 64);
    r.n = (int)(hi - lo);
    return true;
}

// Keys or values, head, sequence and block of the sequence's of this workgroup; slots: blocks that each sequence may touch,
// or places of all (`packed`).
struct KvPlace {
    bool keys;
    int h, s, slot;
};

__device__ __forceinline__ KvPlace kv_place(const ba_kv_args& a, int slots, int packed) {
    unsigned id = blockIdx.x;
    KvPlace r;
    r.keys = (id & 1) == 0;
    id >>= 1;
    r.h = (int)(id % (unsigned)a.heads);
    id /= (unsigned)a.heads;
    r.s = (int)(id / (unsigned)slots);
    r.slot = (int)(id % (unsigned)slots);
    // n rows touch (n + 62) / 64 + 1 blocks at most, which is n / 64 + 2 or less
    if (packed) r.s = seq_of_place(a.offsets, a.n_seqs, a.n_rows, 1, 64, 2, (unsigned)r.slot, r.slot);
    return r;
}

__device__ __forceinline__ bool kv_there(const ba_kv_args& a, const KvShare& r) { return r.page >= 0 && r.page < a.n_blocks; }

__device__ __forceinline__ uint32_t f32_bits(float x) { return __builtin_bit_cast(uint32_t, x); }

// the factor for values of at most amax (given as its bits)
template <int KT>
__device__ __forceinline__ float kv_fit(uint32_t bits) {
    if (bits >= 0x7f800000u) return __builtin_nanf("");
    if (KT == BA_FP8) {
        const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);       // 448 = 1.75 * 2^8
        if (e > 60) return __builtin_nanf("");
        return __builtin_bit_cast(float, (uint32_t)((e < -60 ? -60 : e) + 127) << 23);
    }
    const float f = fmaxf(__builtin_bit_cast(float, bits) / 127.0f, 0x1p-60f);
    return f > 0x1p60f ? __builtin_nanf("") : f;
}

template <int KT>
__device__ __forceinline__ uint32_t kv_code4(float a, float b, float c, float d) {
    if (KT == BA_FP8) {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
    }
    // 1.5 * 2^23 + x is x rounded to a whole number, ties to even, with its low byte last; |x| is at most 127 by the
    // choice of the factor
    auto one = [](float x) { return __builtin_bit_cast(uint32_t, x + 12582912.0f); };
    const uint32_t lo = __builtin_amdgcn_perm(one(b), one(a), 0x0c0c0400u), hi = __builtin_amdgcn_perm(one(d), one(c), 0x0c0c0400u);
    return hi << 16 | lo;
}

template <int KT>
__device__ __forceinline__ void kv_values4(uint32_t w, float (&v)[4]) {
    if (KT == BA_FP8) {
        typedef float f2 __attribute__((ext_vector_type(2)));
        const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        v[0] = lo.x; v[1] = lo.y; v[2] = hi.x; v[3] = hi.y;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (float)(int8_t)(w >> (8 * i));
    }
}

// codes of the tokens before `at` in a word that starts with token `first`, made anew with another factor
template <int KT>
__device__ __forceinline__ uint32_t kv_recode4(uint32_t w, float ratio, int keep) {
    float v[4];
    kv_values4<KT>(w, v);
    const uint32_t n = kv_code4<KT>(v[0] * ratio, v[1] * ratio, v[2] * ratio, v[3] * ratio);
    const uint32_t mask = keep >= 4 ? ~0u : keep <= 0 ? 0u : (1u << (8 * keep)) - 1u;
    return (n & mask) | (w & ~mask);
}

template <typename T, int V>
__device__ __forceinline__ void load_row(const T* p, bool wide, float (&v)[V]) {
    if (wide) {
        load_vec<T, V>(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (float)p[i];
    }
}

// the codes of a values block into the tile
template <int D>
__device__ __forceinline__ void load_tile(const uint8_t* base, uint32_t* tile) {
#pragma unroll
    for (int i = 0; i < (4 * D + KV_T - 1) / KV_T; ++i) {
        const int q = threadIdx.x + i * KV_T;
        if (4 * D % KV_T != 0 && q >= 4 * D) break;
        const uint4 w = ((const uint4*)base)[q];
        uint32_t* t = tile + q / 4 * (KV_ROW / 4) + q % 4 * 4;
        t[0] = w.x; t[1] = w.y; t[2] = w.z; t[3] = w.w;
    }
}

// KEYS: a thread takes 8 elements of a token (UNITS times); values: 4 or 8 elements of 4 tokens.
template <int D, int KT, typename T, bool KEYS>
__device__ void kv_write_block(const ba_kv_args& a, const KvShare& sh, int h, bool wide, uint32_t* tile, uint32_t* red) {
    // 8 values of 4 tokens where that keeps most threads busy (rows of 96 to int8 18.7 -> 16.3 us, of 128 27.8 -> 24; of 64 17.8 -> 18.3)
    constexpr int W = KEYS || D >= 96 ? 8 : 4, ROWS = KEYS ? 1 : 4, PER_ROW = D / W;
    constexpr int N = PER_ROW * (64 / ROWS), UNITS = (N + KV_T - 1) / KV_T;
    const int tid = threadIdx.x;
    const T* x = (const T*)(KEYS ? a.rk : a.rv);
    const int st = (int)(KEYS ? a.rk_st : a.rv_st);         // below 2^31: a row's address is one multiply-add
    x += sh.row * st + h * (KEYS ? a.rk_sh : a.rv_sh);
    // tokens of a unit are block places sh.at + t; a values unit starts at a place that is a multiple of 4
    const int at4 = KEYS ? sh.at : sh.at & ~3;
    float v[UNITS][ROWS][W];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
        const int u = tid + i * KV_T, e = u % PER_ROW * W, place = at4 + u / PER_ROW * ROWS;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int t = place + r - sh.at;
            if (u < N && t >= 0 && t < sh.n) {
                load_row<T, W>(x + (int64_t)t * st + e, wide, v[i][r]);
            } else {
#pragma unroll
                for (int j = 0; j < W; ++j) v[i][r][j] = 0.0f;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < UNITS; ++i)
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int j = 0; j < W; ++j) top = max(top, f32_bits(v[i][r][j]) & 0x7fffffffu);
    // the rows were under way before the block's number was needed
    if (!kv_there(a, sh)) return;
    uint8_t* base = (uint8_t*)(KEYS ? a.k : a.v) + (sh.page * a.heads + h) * (int64_t)(64 * D);
    float* factor = a.scales + (sh.page * a.heads + h) * 2 + (KEYS ? 0 : 1);
    const float old = sh.at ? *factor : 0.0f;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m));
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
    top = max(max(red[0], red[1]), max(red[2], red[3]));
    float f = kv_fit<KT>(top);
    if (sh.at && !(f > old)) f = f == f ? old : f;                   // a NaN factor stays, and a new NaN wins
    const bool poisoned = f != f;
    const float inv = poisoned ? 0.0f : 1.0f / f;
    const bool again = sh.at && f > old;
    const float ratio = again ? old / f : 1.0f;
    if (tid == 0 && (sh.at == 0 || f != old)) *factor = f;
    if (poisoned) {
#pragma unroll
        for (int i = 0; i < UNITS; ++i)
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
#pragma unroll
                for (int j = 0; j < W; ++j) v[i][r][j] = 0.0f;
    }

    if constexpr (KEYS) {
        if (again)
            for (int q = tid; q < sh.at * (D / 4); q += KV_T) {
                uint32_t* w = (uint32_t*)base + q;
                *w = kv_recode4<KT>(*w, ratio, 4);
            }
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const int u = tid + i * KV_T, t = u / PER_ROW;
            if (t >= sh.n) continue;
            const float* y = v[i][0];
            uint2 c;
            c.x = kv_code4<KT>(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
            c.y = kv_code4<KT>(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv);
            *(uint2*)(base + (sh.at + t) * D + u % PER_ROW * W) = c;
        }
        return;
    }
    // a few tokens that need no new codes beside them: bytes
    if (sh.n < KV_FEW && !again) {
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const int u = tid + i * KV_T, e = u % PER_ROW * W, place = at4 + u / PER_ROW * ROWS;
            if (u >= N || place >= sh.at + sh.n) continue;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const uint32_t c = kv_code4<KT>(v[i][0][j] * inv, v[i][1 % ROWS][j] * inv, v[i][2 % ROWS][j] * inv,
                                                v[i][3 % ROWS][j] * inv);
#pragma unroll
                for (int r = 0; r < ROWS; ++r)
                    if (place + r >= sh.at && place + r < sh.at + sh.n) base[(e + j) * 64 + place + r] = (uint8_t)(c >> (8 * r));
            }
        }
        return;
    }
    // through the tile: row d has the 64 tokens of element d
    const bool whole = sh.at == 0 && sh.n == 64;
    if (!whole) {
        load_tile<D>(base, tile);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
        const int u = tid + i * KV_T, e = u % PER_ROW * W, place = at4 + u / PER_ROW * ROWS;
        if (u >= N || place >= sh.at + sh.n) continue;
        const int lo = sh.at > place ? sh.at - place : 0, hi = sh.at + sh.n - place;
        const uint32_t mask = (hi >= 4 ? ~0u : (1u << (8 * hi)) - 1u) & ~((1u << (8 * lo)) - 1u);
#pragma unroll
        for (int j = 0; j < W; ++j) {
            uint32_t* w = tile + (e + j) * (KV_ROW / 4) + place / 4;
            const uint32_t c = kv_code4<KT>(v[i][0][j] * inv, v[i][1 % ROWS][j] * inv, v[i][2 % ROWS][j] * inv,
                                            v[i][3 % ROWS][j] * inv);
            *w = mask == ~0u ? c : (c & mask) | (*w & ~mask);
        }
    }
    __syncthreads();
    for (int q = tid; q < D * 4; q += KV_T) {
        const uint32_t* t = tile + q / 4 * (KV_ROW / 4) + q % 4 * 4;
        uint32_t w[4] = {t[0], t[1], t[2], t[3]};
        if (again)
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = kv_recode4<KT>(w[j], ratio, sh.at - (q % 4 * 16 + 4 * j));
        ((uint4*)base)[q] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <int D, int KT, typename T>
__global__ void __launch_bounds__(KV_T) k_kv_write(ba_kv_args a, int slots, int packed, int wide) {
    __shared__ uint32_t tile[D * (KV_ROW / 4)];
    __shared__ uint32_t red[4];
    const KvPlace at = kv_place(a, slots, packed);
    KvShare sh;
    if (at.slot < 0 || !kv_share(a, at.s, at.slot, sh)) return;
    if (at.keys) kv_write_block<D, KT, T, true>(a, sh, at.h, wide != 0, tile, red);
    else kv_write_block<D, KT, T, false>(a, sh, at.h, wide != 0, tile, red);
}

template <int D, int KT, typename T>
__global__ void __launch_bounds__(KV_T) k_kv_read(ba_kv_args a, int slots, int packed, int wide) {
    __shared__ uint32_t tile[D * (KV_ROW / 4)];
    const KvPlace at = kv_place(a, slots, packed);
    const bool keys = at.keys;
    const int h = at.h, s = at.s, slot = at.slot, tid = threadIdx.x;
    if (slot < 0) return;
    KvShare sh;
    bool held = kv_share(a, s, slot, sh);
    if (held) {
        sh.page = kv_block((int32_t)sh.page);
        held = kv_there(a, sh);
    }
    T* y = (T*)(keys ? a.rk : a.rv);
    const int st = (int)(keys ? a.rk_st : a.rv_st);         // below 2^31: a row's address is one multiply-add
    y += h * (keys ? a.rk_sh : a.rv_sh);
    if (!held) {                                             // rows of the call that no block holds are zeros
        int64_t row0 = (int64_t)s * a.rows_per_seq, count = a.rows_per_seq;
        if (a.offsets) { row0 = a.offsets[s]; count = (int64_t)a.offsets[s + 1] - row0; }
        if (row0 < 0) return;
        count = count < a.max_rows ? count : a.max_rows;
        count = count < a.n_rows - row0 ? count : a.n_rows - row0;
        const int64_t start = a.starts[s], off = start < 0 ? 0 : start % 64;
        const int64_t lo = slot ? (int64_t)slot * 64 - off : 0, end = (int64_t)slot * 64 + 64 - off;
        const int64_t hi = count < end ? count : end;
        for (int64_t q = lo * D + tid; q < hi * D; q += KV_T) y[(row0 + q / D) * st + q % D] = (T)0.0f;
        return;
    }
    y += sh.row * st;
    const uint8_t* base = (const uint8_t*)(keys ? a.k : a.v) + (sh.page * a.heads + h) * (int64_t)(64 * D);
    const float f = a.scales[(sh.page * a.heads + h) * 2 + (keys ? 0 : 1)];
    // W elements to a store of 16 bytes where there is work for all threads
    constexpr int W = sizeof(T) == 2 ? 8 : 4, WV = D >= 128 ? W : 4;
    auto store = [&](T* p, const auto& v) {
        constexpr int N = sizeof(v) / sizeof(float);
        if (wide) {
            store_vec<T, N>(p, v);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) p[j] = (T)v[j];
        }
    };
    if (keys) {
        constexpr int UNITS = (64 * (D / W) + KV_T - 1) / KV_T;
        uint32_t w[UNITS][W / 4];
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {                    // all loads before the first store
            const int q = tid + i * KV_T;
            if (q >= sh.n * (D / W)) break;
#pragma unroll
            for (int j = 0; j < W / 4; ++j) w[i][j] = ((const uint32_t*)base)[(sh.at * (D / W) + q) * (W / 4) + j];
        }
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const int q = tid + i * KV_T;
            if (q >= sh.n * (D / W)) break;
            float v[W];
#pragma unroll
            for (int j = 0; j < W; j += 4) {
                float x[4];
                kv_values4<KT>(w[i][j / 4], x);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[j + k] = x[k] * f;
            }
            store(y + (int64_t)(q / (D / W)) * st + q % (D / W) * W, v);
        }
        return;
    }
    load_tile<D>(base, tile);
    __syncthreads();
    for (int u = tid; u < 16 * (D / WV); u += KV_T) {        // WV elements of 4 tokens
        const int e = u % (D / WV) * WV, place = u / (D / WV) * 4;
        if (place + 4 <= sh.at || place >= sh.at + sh.n) continue;
        float v[WV][4];
#pragma unroll
        for (int j = 0; j < WV; ++j) kv_values4<KT>(tile[(e + j) * (KV_ROW / 4) + place / 4], v[j]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int t = place + r - sh.at;
            if (t < 0 || t >= sh.n) continue;
            float o[WV];
#pragma unroll
            for (int j = 0; j < WV; ++j) o[j] = v[j][r] * f;
            store(y + (int64_t)t * st + e, o);
        }
    }
}

template <int D, int KT, typename T>
static int launch_kv(const ba_kv_args& a, bool write, int slots, bool packed, unsigned nb, hipStream_t st) {
    const int64_t s[4] = {a.rk_st, a.rk_sh, a.rv_st, a.rv_sh};
    // a thread moves 8 elements at a time at most
    bool wide = (uintptr_t)a.rk % 16 == 0 && (uintptr_t)a.rv % 16 == 0;
    for (int i = 0; i < 4; ++i) wide = wide && s[i] % 8 == 0;
    if (write) hipLaunchKernelGGL((k_kv_write<D, KT, T>), dim3(nb), dim3(KV_T), 0, st, a, slots, (int)packed, (int)wide);
    else hipLaunchKernelGGL((k_kv_read<D, KT, T>), dim3(nb), dim3(KV_T), 0, st, a, slots, (int)packed, (int)wide);
    BA_LAUNCHED();
    return BA_OK;
}

static int kv_call(const ba_kv_args* args, void* stream, bool write) {
    clear_error();
    BA_REQUIRE(args != nullptr, "null args");
    const ba_kv_args& a = *args;
    BA_REQUIRE(a.n_blocks >= 0 && a.n_blocks <= KV_KEPT && a.heads >= 1 && a.heads <= 65536 && a.n_seqs >= 0 && a.n_pages >= 0, "cache: bad sizes");
    BA_REQUIRE(a.dim == 32 || a.dim == 64 || a.dim == 96 || a.dim == 128 || a.dim == 256,
               "cache: head size must be 32, 64, 96, 128 or 256");
    BA_REQUIRE(a.bits == BA_FP8 || a.bits == BA_INT8, "cache: bits must be 0 (e4m3) or 1 (int8)");
    BA_REQUIRE(a.dtype >= 0 && a.dtype <= 2, "cache: rows must be fp32, fp16 or bf16");
    BA_REQUIRE(a.n_rows >= 0 && a.rows_per_seq >= 0 && a.max_rows >= 0 && a.n_rows < (int64_t)1 << 31 && a.max_rows < (int64_t)1 << 31 &&
                   a.rows_per_seq < (int64_t)1 << 31, "cache: bad sizes");
    if (a.n_rows == 0 || a.n_seqs == 0 || a.max_rows == 0) return BA_OK;
    BA_REQUIRE(a.starts && a.rk && a.rv, "null pointer");
    BA_REQUIRE((a.n_pages == 0 || a.pages) && (a.n_blocks == 0 || (a.k && a.v && a.scales)), "null pointer");
    BA_REQUIRE((uintptr_t)a.k % 16 == 0 && (uintptr_t)a.v % 16 == 0, "cache: k and v must be aligned to 16 bytes");
    const int64_t strides[4] = {a.rk_st, a.rk_sh, a.rv_st, a.rv_sh};
    for (int i = 0; i < 4; ++i)
        BA_REQUIRE(strides[i] > -((int64_t)1 << 31) && strides[i] < (int64_t)1 << 31, "cache: strides of rows and heads must be below 2^31");
    int64_t slots = (a.max_rows + 62) / 64 + 1, per_slot = (int64_t)a.n_seqs * a.heads;
    // a launch has less than 2^32 threads
    const int64_t most = ((int64_t)1 << 23) - 1;
    const bool packed = a.offsets && slots > most / per_slot;
    if (packed) {
        slots = a.n_rows / 64 + 2 * (int64_t)a.n_seqs;
        per_slot = a.heads;
    }
    BA_REQUIRE(slots <= most / per_slot, "cache: too many blocks for a call");
    const unsigned nb = (unsigned)(slots * per_slot * 2);
    hipStream_t st = (hipStream_t)stream;
#define BA_KV_D(D, KT, T) case D: return launch_kv<D, KT, T>(a, write, (int)slots, packed, nb, st);
#define BA_KV_ALL(KT, T) \
    switch (a.dim) { BA_KV_D(32, KT, T) BA_KV_D(64, KT, T) BA_KV_D(96, KT, T) BA_KV_D(128, KT, T) BA_KV_D(256, KT, T) }
    if (a.bits == BA_FP8) {
        if (a.dtype == BA_F32) { BA_KV_ALL(BA_FP8, float) }
        else if (a.dtype == BA_F16) { BA_KV_ALL(BA_FP8, _Float16) }
        else { BA_KV_ALL(BA_FP8, __bf16) }
    } else {
        if (a.dtype == BA_F32) { BA_KV_ALL(BA_INT8, float) }
        else if (a.dtype == BA_F16) { BA_KV_ALL(BA_INT8, _Float16) }
        else { BA_KV_ALL(BA_INT8, __bf16) }
    }
#undef BA_KV_ALL
#undef BA_KV_D
    return BA_ERR_UNSUPPORTED;
}

}  // namespace ba

using namespace ba;

extern "C" int ba_kv_write(const ba_kv_args* args, void* stream) { return kv_call(args, stream, true); }
extern "C" int ba_kv_read(const ba_kv_args* args, void* stream) { return kv_call(args, stream, false); }
