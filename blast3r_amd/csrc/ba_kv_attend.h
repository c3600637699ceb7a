// Attention over the 8-bit key/value cache.
//
// For a row of queries q and the keys j that it sees,  o = sum_j p_j v_j / sum_j p_j,  p_j = exp(c q.k_j - m):
// one pass over the cache with a running reference m, so that the scores never leave the registers.
//
// Rows of a wave are query rows that share a cache head (the tokens of a sequence times the query heads of that
// cache head); it walks over blocks of 64 tokens with two matrix products each, laid out so that the weights
// never change lanes:
//   scores   S^T = K Q^T: lane (n, g) of COLS x NG holds 8-element pieces of key rows and of query row n.  Which
//            token a key row of the product stands for is free, and is chosen so that
//   products O^T = V^T P^T: the lane's scores are those of 64 / NG consecutive tokens for query row n, which is
//            the layout of this product's second operand (P) as it stands; the values, kept as (dim, 64), are
//            consecutive bytes.
// Codes become fp16, which holds each of them exactly (bf16 would too, but has 8 bits for the weights); queries
// are scaled by a power of two of their row to fp16, exactly for bf16 and fp16 queries down to 2^-28 of the
// row's largest element; sums are fp32.
//
// Factors: a block's key factor goes into the constant c, its value factor into the exponent: with z = c q.k
// and lv = log2(value factor), m follows z + lv, so that the weights exp2(z + lv - m) that meet the codes of
// the values fit fp16 whatever the factors are, and the denominator adds their sums divided by the value
// factor.  Weights are rounded to fp16: 11 bits, an eighth of the error of rounding a bf16 output, but as much
// as rounding an fp16 one.  For fp16 outputs (HALF) the rounded weights make up the denominator too, so that a
// row that one key dominates is exact (errors against 64 bits 1.0 to 1.3 times those of rounding the output,
// 1.2 to 1.4 without; 3% of the time of k_kv_attend_tile at 128 elements); for bf16 the unrounded ones do.
// Weights of a block whose values are small beside others' (by AT_LOW) may vanish in fp16 and still count in
// the denominator: its sums are taken before rounding in any case.  m is moved only when a weight nears
// fp16's end; until then nothing is rescaled.  log2 and reciprocal of a value factor are the hardware's, right to the
// last place of fp32 or so: with |lv| up to 60 a block's weights are off by 3e-6 in all, against fp16's 5e-4 of each.
//
// Two kernels (figures of the plain form; what the other forms add and take is in ba_kv_scored.hip):
//   k_kv_attend       up to 32 rows: the waves of a workgroup have the same rows and split the blocks, codes go
//                     from memory to registers without LDS, and the waves' sums are joined at the end.  Bound by
//                     memory: a query over 192000 tokens of 16 heads of 64 (393 MB) takes 70 to 74 us, 5.3 to 5.6 TB/s;
//                     48 sequences of up to 8192 tokens, 8 heads of 128 (417 MB), 89 to 92 us, 4.6 TB/s (a large copy:
//                     4.8); 16 sequences of 8192 tokens with 2, 5 and 32 rows (269 MB) 50, 50 and 56 us with the join.
//   k_kv_attend_tile  more rows: the waves split the rows and share blocks that are converted to fp16 once, in LDS.
//                     Bound by the vector and matrix units together, and by power (the clock falls to 2.0 - 2.2
//                     GHz): 2 x 2048 rows over 16384 tokens, 32 heads of 128: 1015 to 1040 us, 1.0 PFLOP/s (a large fp16
//                     matrix product on this card: 1.09); of 64: 565 to 580 us, 0.9 PFLOP/s, where the exponentials alone
//                     take as long as half of the products; of 32: 490 us, 0.5 PFLOP/s; of 96: 900, 0.86; 16 heads of 256:
//                     1240, 0.83.  Where tiles are few or of different lengths workgroups are what is missing: a prompt
//                     of 2048 rows into an empty cache takes 70 us of 32, 768 rows over 768 tokens 24 us of 2.
// Where rows are few the blocks of a sequence are further cut into n_splits parts, whose sums k_kv_join adds in
// order (5 us for 16 rows of 24 parts, 10 us for 12288 rows of 10).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

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
#define AT_MIN_BLOCKS 16     // a part has at least so many blocks: below that the join costs more than it saves (a query over
                             // 777 tokens 12 us in one part, 18 in two; over 8192 tokens 18.5 in 8 parts, 17.8 in 16;
                             // measured with k_kv_attend only)

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

// What a kernel does with scores and with what rows see.  Few rows are bound by memory, and one form decides as it runs; the
// tiles' exponents stand between matrix products, instruction by instruction, and each has a kernel of its own.
//   AT_PLAIN   softmax(scale q.k) over the tokens up to a row's own (causal) and in its window
//   AT_MASKS   a row's tokens are [lo, hi) and those below pre (AtRow); a launch may take some of the lists' blocks only, and
//              the rows of all sequences together
//   AT_SLOPES  the same, less slope |position - token| in each score
//   AT_CAPPED  the same as AT_MASKS, with cap tanh(score / cap) in the place of each score
//   AT_BOTH    capped, then less the slopes' part
//   AT_ANY     what the call asks for
enum { AT_PLAIN = 0, AT_MASKS = 1, AT_SLOPES = 2, AT_CAPPED = 3, AT_BOTH = 4, AT_ANY = 5 };
constexpr bool at_slopes(int mode) { return mode == AT_SLOPES || mode == AT_BOTH || mode == AT_ANY; }
constexpr bool at_caps(int mode) { return mode == AT_CAPPED || mode == AT_BOTH || mode == AT_ANY; }

// what differs between the workgroups of a launch that is not plain
struct AtPart {
    int blk_lo, blk_hi;      // the blocks of the lists that they take
    int part0, parts;        // they write the parts [part0, part0 + parts) of the n_splits
    int least;               // blocks of a part at least
    int stacked;             // their rows are those of all sequences, and a workgroup's list is that of its row that sees furthest
    int tiles, packed;       // their grid (AtGrid), and
    unsigned first, wgs;     // which of the launch's they are
};

// of a launch that is not plain
struct AtMore {
    const float* slopes;     // of the query heads, or NULL
    const int32_t* prefix;   // of the sequences, or NULL
    const int32_t* since;    // of the rows, or NULL
    const int32_t* until;
    float cap;
    int mix;                 // rows of tiles (a head, a part) that each XCD has whole, 0 where it has none so, -1: tiles are alike
    AtPart p;
};

template <int MODE> struct AtArgs {
    ba_kv_attend_args a;
    AtMore m;
};
template <> struct AtArgs<AT_PLAIN> {
    ba_kv_attend_args a;
};
// Few rows: shared blocks and the sequences' own are one launch, whose later workgroups (`after`) run beside the others where
// these leave the CUs room (64 tokens over 16384 shared and up to 512 of their own 60 -> 52 us, 16 over 8192 and 1000 39 -> 26).
template <> struct AtArgs<AT_ANY> {
    ba_kv_attend_args a;
    AtMore m;
    AtPart after;
};

// the arguments of this workgroup
template <int MODE>
__device__ __forceinline__ decltype(auto) at_args(const AtArgs<MODE>& x) {
    if constexpr (MODE == AT_ANY) {
        // each field chosen by itself: of a copied struct the compiler chooses addresses, and loads wait for loads (0.4 us a call)
        const AtPart &l = x.m.p, &r = x.after;
        const bool after = blockIdx.x >= l.wgs;
        AtArgs<MODE> y = x;
        y.m.p = {after ? r.blk_lo : l.blk_lo, after ? r.blk_hi : l.blk_hi, after ? r.part0 : l.part0, after ? r.parts : l.parts,
                 after ? r.least : l.least, after ? r.stacked : l.stacked, after ? r.tiles : l.tiles, after ? r.packed : l.packed,
                 after ? r.first : l.first, after ? r.wgs : l.wgs};
        return y;
    } else {
        return (x);
    }
}

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

// What a sequence of the call has: its rows and its tokens.
struct AtSeq {
    int64_t row0;
    int len;                 // tokens within its block list
    int first;               // position of its first row: that of all its rows and tokens, there or not
    int rows;                // of its rows, those within max_rows
};

__device__ __forceinline__ AtSeq at_seq(const ba_kv_attend_args& a, int s) {
    int64_t row0 = (int64_t)s * a.rows_per_seq, n = a.rows_per_seq;
    if (a.offsets) {
        row0 = a.offsets[s];
        n = (int64_t)a.offsets[s + 1] - row0;
    }
    if (row0 < 0 || row0 > a.n_rows || n < 0) { row0 = 0; n = 0; }
    int64_t len = a.lengths[s];
    len = len < 0 ? 0 : len;
    const int first = (int)(len - n);
    n = n < a.n_rows - row0 ? n : a.n_rows - row0;
    const int64_t most = (int64_t)a.n_pages * 64;
    return {row0, (int)(len < most ? len : most), first, (int)(n < a.max_rows ? n : a.max_rows)};
}

// The tile, part, head and sequence of this workgroup; n_tiles: tiles of each sequence, or places of all (`packed`).
struct AtPlace {
    int tile, sp, kh, s;
};

// Later rows see more (their tiles come first below), and workgroups of one CU should see as much together as those of another:
// tiles of all heads that an XCD has go by their length, and every other 32 of them, which its CUs take in turn, from the
// shortest (6144 rows of frames over 12288 tokens, 16 heads of 64: 312 -> 289 us; prompts of 2048 for 4 sequences into an empty
// cache, 32 heads on 8: 149 -> 131; 8 of 768 after as many 126 -> 115).  Tiles that are alike, and few rows, are better off in
// their own order, where those of one head read the same blocks at the same time (391 against 400, 80 against 94).
__device__ __forceinline__ unsigned at_turn(int mix, int n_tiles) {
    const unsigned nb = gridDim.x, x = blockIdx.x % BA_N_XCD, q = nb / BA_N_XCD, r = nb % BA_N_XCD;
    const unsigned n = q + (x < r ? 1u : 0u), first = x * q + (x < r ? x : r);
    unsigned k = blockIdx.x / BA_N_XCD;
    if ((k & 32u) && (k | 31u) < n) k ^= 31u;
    if (mix > 1) {
        const unsigned rank = k / (unsigned)mix;
        k = (k - rank * (unsigned)mix) * (unsigned)n_tiles + rank;
    }
    return first + k;
}

template <int MODE>
__device__ __forceinline__ AtPlace at_place(const AtArgs<MODE>& x, int rows, int n_tiles, int packed) {
    const ba_kv_attend_args& a = x.a;
    unsigned id = xcd_block(blockIdx.x, gridDim.x), parts = (unsigned)a.n_splits;
    if constexpr (MODE == AT_ANY) {
        n_tiles = x.m.p.tiles;
        packed = x.m.p.packed;
        id = xcd_block(blockIdx.x - x.m.p.first, x.m.p.wgs);
        parts = (unsigned)x.m.p.parts;
    } else if constexpr (MODE != AT_PLAIN) {
        parts = (unsigned)x.m.p.parts;
        if (x.m.mix >= 0) id = at_turn(x.m.mix, n_tiles);
    }
    AtPlace r;
    r.tile = (int)(id % (unsigned)n_tiles);
    id /= (unsigned)n_tiles;
    r.sp = (int)(id % parts);
    id /= parts;
    r.kh = (int)(id % (unsigned)a.heads);
    r.s = (int)(id / (unsigned)a.heads);
    if (MODE != AT_PLAIN) r.tile = n_tiles - 1 - r.tile;     // later rows see more: the longest tiles first
    if (packed) r.s = seq_of_place(a.offsets, a.n_seqs, a.n_rows, a.q_heads / a.heads, rows, 1, (unsigned)r.tile, r.tile);
    return r;
}

// the sequence of a row: the last whose first row is not after it
__device__ __forceinline__ int seq_of_row(const ba_kv_attend_args& a, int64_t row) {
    if (!a.offsets) {
        const unsigned s = (unsigned)row / (unsigned)a.rows_per_seq;
        return s < (unsigned)a.n_seqs ? (int)s : a.n_seqs - 1;
    }
    int s = 0, e = a.n_seqs;
    while (e - s > 1) {
        const int c = (s + e) >> 1;
        if (a.offsets[c] <= row) s = c; else e = c;
    }
    return s;
}

// Blocks [lo, hi) that rows [row, row + rows) (of the sequence's rows * group) see, cut into parts of `per` blocks.
struct AtBlocks {
    int lo, hi, per;
};

__device__ __forceinline__ AtBlocks at_blocks(const ba_kv_attend_args& a, const AtSeq& q, int group, int row, int rows) {
    const int all = q.rows * group, last = row + rows < all ? row + rows : all;
    if (row >= last) return {0, 0, 1};
    const int p0 = q.first + (int)((unsigned)row / (unsigned)group), p1 = q.first + (int)((unsigned)(last - 1) / (unsigned)group);
    const int keys = a.causal && p1 < q.len ? p1 + 1 : q.len;
    const int64_t from = a.window > 0 ? p0 - a.window + 1 : 0;
    const int first = from < 0 ? 0 : from < q.len ? (int)from : q.len;
    if (keys <= first) return {0, 0, 1};
    const int b0 = first / 64, b1 = (keys + 63) / 64, per = (b1 - b0 + a.n_splits - 1) / a.n_splits;
    return {b0, b1, per < AT_MIN_BLOCKS ? AT_MIN_BLOCKS : per};
}

// Part sp of them.
__device__ __forceinline__ void at_part(const AtBlocks& b, int sp, int& lo, int& hi) {
    const int64_t x = b.lo + (int64_t)sp * b.per;
    lo = x < b.hi ? (int)x : b.hi;
    hi = lo + b.per < b.hi ? lo + b.per : b.hi;
}

// What a row sees when it is not plain: tokens below pre, and [lo, hi) where that is not empty (else lo is AT_NEVER and hi 0).
struct AtRow {
    int pos, lo, hi, pre;
    int seq;                 // its sequence
};
#define AT_NEVER 0x7fffffff

// row i of a sequence's (of all, where they are stacked: one that no sequence has sees nothing)
template <int MODE>
__device__ __forceinline__ AtRow at_row(const AtArgs<MODE>& x, AtSeq q, int s, int64_t i) {
    const ba_kv_attend_args& a = x.a;
    const int64_t row = q.row0 + i;
    if (x.m.p.stacked) {
        s = seq_of_row(a, row);
        q = at_seq(a, s);
        i = row - q.row0;
        if (i < 0 || i >= q.rows) return {0, AT_NEVER, 0, 0, s};
    }
    const int64_t pos = (int64_t)q.first + i, since = x.m.since ? x.m.since[row] : 0, until = x.m.until ? x.m.until[row] : q.len;
    const int64_t from = a.window > 0 ? pos - a.window + 1 : 0, end = a.causal ? pos + 1 : q.len;
    const int64_t lo = since > from ? since : from, hi = until < end ? until : end;
    const int l = (int)(lo < 0 ? 0 : lo), h = (int)(hi < q.len ? hi : q.len);
    const int pre = x.m.prefix ? x.m.prefix[s] : 0;
    return {(int)pos, h > l ? l : AT_NEVER, h > l ? h : 0, pre < 0 ? 0 : pre < q.len ? pre : q.len, s};
}

// Distance that a row's biases are measured from: that of the token it sees whose bias is the largest.  Far tokens' biases
// are large numbers that the softmax takes from one another; what matters of them is small.
__device__ __forceinline__ int at_anchor(const AtRow& r, float slope) {
    const bool main = r.hi > r.lo, pre = r.pre > 0;
    int d;
    auto far = [&](int j) { return r.pos < j ? j - r.pos : r.pos - j; };
    if (slope >= 0.0f) {
        d = AT_NEVER;
        if (main) d = r.pos < r.lo ? r.lo - r.pos : r.pos >= r.hi ? r.pos - r.hi + 1 : 0;
        if (pre) d = min(d, r.pos < 0 ? -r.pos : r.pos >= r.pre ? r.pos - r.pre + 1 : 0);
        return d == AT_NEVER ? 0 : d;
    }
    d = 0;
    if (main) d = max(far(r.lo), far(r.hi - 1));
    if (pre) d = max(d, max(far(0), far(r.pre - 1)));
    return d;
}

// The tokens [at, at + 32) that a row sees, a bit each; a score whose bit is not set is hidden (two instructions a score where
// comparisons take five).
__device__ __forceinline__ uint32_t at_bits(const AtRow& r, int at) {
    auto below = [](int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; };
    return below(r.pre - at) | (below(r.hi - at) & ~below(r.lo - at));
}
__device__ __forceinline__ float at_hidden(float score, uint32_t bits, int t) {
    const uint32_t keep = (uint32_t)((int32_t)(bits << (31 - t)) >> 31);
    return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, score) & keep) | (0xff800000u & ~keep));
}

// the smallest and largest of what rows see
struct AtSpan {
    int lo0, lo1, hi0, hi1, pre0, pre1, pos0, pos1;
};

template <int N, int COLS>
__device__ __forceinline__ AtSpan at_span(const AtRow (&r)[N]) {
    AtSpan s = {r[0].lo, r[0].lo, r[0].hi, r[0].hi, r[0].pre, r[0].pre, r[0].pos, r[0].pos};
    auto more = [&](int lo0, int lo1, int hi0, int hi1, int pre0, int pre1, int pos0, int pos1) {
        s.lo0 = min(s.lo0, lo0);
        s.lo1 = max(s.lo1, lo1);
        s.hi0 = min(s.hi0, hi0);
        s.hi1 = max(s.hi1, hi1);
        s.pre0 = min(s.pre0, pre0);
        s.pre1 = max(s.pre1, pre1);
        s.pos0 = min(s.pos0, pos0);
        s.pos1 = max(s.pos1, pos1);
    };
#pragma unroll
    for (int c = 1; c < N; ++c) more(r[c].lo, r[c].lo, r[c].hi, r[c].hi, r[c].pre, r[c].pre, r[c].pos, r[c].pos);
#pragma unroll
    for (int k = 1; k < COLS; k <<= 1)
        more(__shfl_xor(s.lo0, k), __shfl_xor(s.lo1, k), __shfl_xor(s.hi0, k), __shfl_xor(s.hi1, k), __shfl_xor(s.pre0, k),
             __shfl_xor(s.pre1, k), __shfl_xor(s.pos0, k), __shfl_xor(s.pos1, k));
    auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    return {one(s.lo0), one(s.lo1), one(s.hi0), one(s.hi1), one(s.pre0), one(s.pre1), one(s.pos0), one(s.pos1)};
}

// The sequence of the row that sees the furthest token, of a wave's rows where these are stacked: it has all blocks that the
// others see of the shared ones (the first sequence may be an empty place of the batch).  Furthest token above, sequence below.
template <int N, int COLS>
__device__ __forceinline__ int64_t at_furthest(const AtRow (&r)[N]) {
    int64_t best = -1;
#pragma unroll
    for (int c = 0; c < N; ++c) {
        const int64_t key = (int64_t)max(r[c].hi, r[c].pre) << 32 | (uint32_t)r[c].seq;
        best = key > best ? key : best;
    }
#pragma unroll
    for (int k = 1; k < COLS; k <<= 1) {
        const int64_t key = (int64_t)__shfl_xor((long long)best, k);
        best = key > best ? key : best;
    }
    return best;
}

// The same of rows i0 .. i1 of a sequence, whose bounds rise with them where neither since nor until says otherwise (rows that
// see nothing widen it, which costs blocks at most).
template <int MODE>
__device__ __forceinline__ AtSpan at_span_of(const AtArgs<MODE>& x, const AtSeq& q, int s, int i0, int i1) {
    const ba_kv_attend_args& a = x.a;
    const int64_t p0 = (int64_t)q.first + i0, p1 = (int64_t)q.first + i1, w = a.window > 0 ? a.window : (int64_t)1 << 40;
    auto at_least0 = [](int64_t v) { return v < 0 ? 0 : (int)v; };
    auto end = [&](int64_t pos) { return a.causal && pos < q.len ? at_least0(pos + 1) : q.len; };
    const int pre = x.m.prefix ? x.m.prefix[s] : 0, p = pre < 0 ? 0 : pre < q.len ? pre : q.len;
    return {at_least0(p0 - w + 1), at_least0(p1 - w + 1), end(p0), end(p1), p, p, (int)p0, (int)p1};
}

// The blocks that a workgroup's rows see in a launch: the first na from a0 on, then those from c0 on, n in all.  Places in
// that row of blocks are what parts are cut by.
struct AtWalk {
    int a0, na, c0, n;
    __device__ __forceinline__ int block(int v) const { return v < na ? a0 + v : c0 + (v - na); }
};

__device__ __forceinline__ AtWalk at_walk(const AtPart& m, int lo, int hi, int pre) {
    AtWalk w;
    w.a0 = m.blk_lo;
    const int a1 = min((int)(((int64_t)pre + 63) / 64), m.blk_hi), c1 = min((int)(((int64_t)hi + 63) / 64), m.blk_hi);
    w.na = max(0, a1 - w.a0);
    w.c0 = max(min(lo / 64, m.blk_hi), w.a0 + w.na);
    w.n = w.na + max(0, c1 - w.c0);
    return w;
}

// the workgroup's rows: of its sequence, or of all
template <int MODE>
__device__ __forceinline__ AtSeq at_rows(const AtArgs<MODE>& x, int s) {
    if constexpr (MODE != AT_PLAIN)
        if (x.m.p.stacked) return {0, 0, 0, (int)x.a.n_rows};
    return at_seq(x.a, s);
}

__device__ __forceinline__ AtBlocks at_cut(const AtWalk& w, const AtPart& m) {
    const int per = (w.n + m.parts - 1) / m.parts;
    return {0, w.n, per < m.least ? m.least : per};
}

// cap tanh(z / cap), as off - 2 cap / (exp(2 z / cap) + 1) with off = cap; `in` brings a score to the exponent of 2.  Off by
// 2^-23 of 2 cap at most.
__device__ __forceinline__ float capped(float score, float in, float out, float off) {
    return fmaf(-out, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(score * in) + 1.0f), off);
}

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
#define AT_MOVE 8.0f          // k_kv_attend moves m when a score passes it by so much (log2)
#define AT_LIFT 6.0f          // weights at m are 2^6: with AT_MOVE at most 2^14, and fp16 is normal down to 2^-20 of m
#define AT_LOW 0.015625f      // a value factor below 2^-6 of the largest so far
#define AT_MOST 32768.0f      // k_kv_attend_tile moves it when a lane's sum of 16 weights passes this: each of them fits fp16

// Query rows row0 .. of a wave (NCB tiles of COLS): their positions, their elements as fp16 (lane (n, g) holds those of
// row n that pair with its pieces of a key) divided by a power of two of the row, and the constant that a score is
// multiplied by before the key factor: softmax scale, log2(e) and that power.
template <int D, int COLS, int NCB>
__device__ __forceinline__ void load_queries(const ba_kv_attend_args& a, const AtSeq& q, int kh, int group, int row0, int all,
                                             int n, int g, bool wide, h8 (&qf)[NCB][D * COLS / 512], float (&qc)[NCB], int (&pos)[NCB]) {
    constexpr int NG = 64 / COLS, KS = D / (8 * NG);
#pragma unroll
    for (int c = 0; c < NCB; ++c) {
        const int r = row0 + c * COLS + n, rc = r < all ? r : all - 1;
        const int i = (int)((unsigned)rc / (unsigned)group);
        const int head = kh * group + rc - i * group;
        pos[c] = q.first + i;
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
}

// What biases take from the logarithm of a row's sum, as its distances are measured from the anchor.
template <int MODE>
__device__ __forceinline__ float lse_shift(const AtArgs<MODE>& x, const AtRow& r, int head) {
    if (!at_slopes(MODE) || !x.m.slopes) return 0.0f;
    const float slope = x.m.slopes[head];
    return slope * (float)at_anchor(r, slope);
}

// The same in two steps, so that the rows are under way while their bounds and the first block are found (documents of 64
// tokens packed into 8192, 32 heads of 128 on 8: 68 -> 54 us).
template <int D, int COLS, int NCB>
__device__ __forceinline__ void fetch_queries(const ba_kv_attend_args& a, const AtSeq& q, int kh, int group, int row0, int all, int n, int g,
                                              bool wide, uint4 (&raw)[NCB][D * COLS / 512]) {
    constexpr int NG = 64 / COLS, KS = D / (8 * NG);
#pragma unroll
    for (int c = 0; c < NCB; ++c) {
        const int r = row0 + c * COLS + n, rc = r < all ? r : all - 1;
        const int i = (int)((unsigned)rc / (unsigned)group);
        const uint16_t* p = (const uint16_t*)a.q + (q.row0 + i) * a.q_st + (kh * group + rc - i * group) * a.q_sh + g * (D / NG);
#pragma unroll
        for (int t = 0; t < KS; ++t) {
            if (wide) {
                raw[c][t] = *(const uint4*)(p + 8 * t);
            } else {
                uint32_t w[4];
                for (int j = 0; j < 4; ++j) w[j] = p[8 * t + 2 * j] | (uint32_t)p[8 * t + 2 * j + 1] << 16;
                raw[c][t] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
}

template <int D, int COLS, int NCB>
__device__ __forceinline__ void shape_queries(const ba_kv_attend_args& a, const uint4 (&raw)[NCB][D * COLS / 512], h8 (&qf)[NCB][D * COLS / 512],
                                              float (&qc)[NCB]) {
    constexpr int NG = 64 / COLS, KS = D / (8 * NG);
#pragma unroll
    for (int c = 0; c < NCB; ++c) {
        uint32_t top = 0;                                    // of the magnitudes, in the bits of either type
#pragma unroll
        for (int t = 0; t < KS; ++t) {
            const uint32_t w[4] = {raw[c][t].x, raw[c][t].y, raw[c][t].z, raw[c][t].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) top = max(top, max(w[j] & 0x7fffu, w[j] >> 16 & 0x7fffu));
        }
#pragma unroll
        for (int m = COLS; m < 64; m <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m));
        auto value = [&](uint32_t bits) {
            return a.dtype == BA_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)bits) : __builtin_bit_cast(float, bits << 16);
        };
        int e = (int)(__builtin_bit_cast(uint32_t, value(top)) >> 23) - 127;     // the row's largest element is in [2^e, 2^(e+1))
        e = e < -100 ? -100 : e > 127 ? 127 : e;
        const float up = __builtin_bit_cast(float, (uint32_t)(14 - e + 127) << 23);
        qc[c] = a.scale * 1.44269504088896341f * __builtin_bit_cast(float, (uint32_t)(e - 14 + 127) << 23);
#pragma unroll
        for (int t = 0; t < KS; ++t) {
            const uint32_t w[4] = {raw[c][t].x, raw[c][t].y, raw[c][t].z, raw[c][t].w};
#pragma unroll
            for (int j = 0; j < 8; ++j) qf[c][t][j] = (_Float16)(value(w[j / 2] >> 16 * (j & 1) & 0xffffu) * up);
        }
    }
}

// The result of a wave's rows, or their partial sums.  A part without blocks leaves its reference only (AT_NONE).
template <int MODE, int D, int COLS, int NCB, typename A>
__device__ __forceinline__ void store_rows(const AtArgs<MODE>& x, const AtSeq& q, int s, int kh, int group, int row0, int all, int sp, bool none,
                                           int n, int g, bool wide, const A (&o)[NCB][D / COLS], const float (&m)[NCB], const float (&l)[NCB]) {
    constexpr int CREG = COLS * COLS / 64, DB = D / COLS;
    typedef Mma<COLS> M;
    const ba_kv_attend_args& a = x.a;
    if constexpr (MODE != AT_PLAIN) sp += x.m.p.part0;
#pragma unroll
    for (int c = 0; c < NCB; ++c) {
        const int r = row0 + c * COLS + n;
        if (r >= all) continue;
        const int i = (int)((unsigned)r / (unsigned)group);
        const int64_t row = q.row0 + i;
        const int head = kh * group + r - i * group;
        if (a.n_splits > 1) {
            float* w = part_sum(a, row, head, sp);
            if (MODE == AT_PLAIN || !none)
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int k = 0; k < CREG; k += 4)
                    *(f4*)(w + d * COLS + M::row(g, k)) = (f4){o[c][d][k], o[c][d][k + 1], o[c][d][k + 2], o[c][d][k + 3]};
            if (g == 0) *part_ref(a, row, head, sp) = make_float2(m[c], l[c]);
            continue;
        }
        const float inv = l[c] == 0.0f ? 0.0f : 1.0f / l[c];         // l is 0 in a row that saw no key
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int k = 0; k < CREG; k += 4)
                store_out4(a, row, head, d * COLS + M::row(g, k),
                           (f4){o[c][d][k] * inv, o[c][d][k + 1] * inv, o[c][d][k + 2] * inv, o[c][d][k + 3] * inv}, wide);
        if (a.lse && g == 0) {
            float lse = l[c] == 0.0f ? -__builtin_inff() : 0.693147180559945309f * (m[c] - AT_LIFT + __builtin_amdgcn_logf(l[c]));
            if constexpr (at_slopes(MODE)) lse -= lse_shift(x, at_row(x, q, s, i), head);
            a.lse[row * a.q_heads + head] = lse;
        }
    }
}

// The slopes of a wave's rows (in units of the exponents, that is times log2(e)) and the anchors of their biases.
template <int MODE, int COLS, int NCB>
__device__ __forceinline__ void load_slopes(const AtArgs<MODE>& x, int kh, int group, int row0, int all, int n, const AtRow (&row)[NCB],
                                            float (&slope)[NCB], int (&anchor)[NCB]) {
#pragma unroll
    for (int c = 0; c < NCB; ++c) {
        slope[c] = 0.0f;
        anchor[c] = 0;
        if (!x.m.slopes) continue;
        const int r = row0 + c * COLS + n, rc = r < all ? r : all - 1;
        const float v = x.m.slopes[kh * group + (int)((unsigned)rc % (unsigned)group)];
        slope[c] = v * 1.44269504088896341f;
        anchor[c] = at_anchor(row[c], v);
    }
}

// waves of a SIMD that the registers are to leave room for
constexpr int at_waves(int d, int cols) { return cols == 16 ? (d <= 64 ? 4 : d <= 128 ? 2 : 1) : d <= 128 ? 2 : 1; }

// Few rows: the waves have the same COLS rows (16 x 16 x 32 products for up to 16, 32 x 32 x 16 for more) and split the
// blocks; every wave reads and converts its own, a block ahead.  8 or 16 waves to a workgroup were no faster on short
// sequences (777 tokens: 8.4 and 9.4 us against 8.5, most of it launch and dependent loads).
template <int MODE, int D, int KT, int COLS, bool HALF>
__global__ void __launch_bounds__(AT_T, at_waves(D, COLS)) k_kv_attend(AtArgs<MODE> args, int n_tiles, int packed, int wide) {
    const auto& x = at_args(args);
    const ba_kv_attend_args& a = x.a;
    typedef Mma<COLS> M;
    typedef typename M::acc acc;
    constexpr int NG = 64 / COLS, NB = NG, CREG = COLS * COLS / 64, TPL = 64 / NG;
    constexpr int KS = D / (8 * NG), DB = D / COLS, PS = TPL / 8, WAVES = AT_T / 64, WK = WAVES, NCB = 1, ROWS = COLS;
    __shared__ float2 ref_sh[WAVES * COLS * NCB];
    __shared__ f4 sum_sh[WAVES / 2 * COLS * NCB * D / 4];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wk = wave;
    const int n = lane % COLS, g = lane / COLS;
    const AtPlace at_wg = at_place(x, ROWS, n_tiles, packed);
    const int tile = at_wg.tile, sp = at_wg.sp, kh = at_wg.kh, s = at_wg.s;
    const int group = a.q_heads / a.heads;
    const AtSeq q = at_rows(x, s);
    const int all = q.rows * group, tile0 = tile * ROWS;
    if (tile < 0 || tile0 >= all) return;
    int lo, hi;
    AtRow row[NCB];
    AtSpan span = {};
    AtWalk walk = {};
    int list = s;                                            // whose list
    auto find_rows = [&] {
        if constexpr (MODE != AT_PLAIN)
#pragma unroll
            for (int c = 0; c < NCB; ++c) {
                const int r = tile0 + c * COLS + n;
                row[c] = at_row(x, q, s, (int)((unsigned)(r < all ? r : all - 1) / (unsigned)group));
            }
    };
    if constexpr (MODE == AT_PLAIN) {
        at_part(at_blocks(a, q, group, tile0, ROWS), sp, lo, hi);
        if (lo >= hi && a.n_splits > 1) return;              // k_kv_join knows which parts there are
    } else {
        if (x.m.since || x.m.until || x.m.p.stacked) {
            find_rows();
            span = at_span<NCB, COLS>(row);
            if (x.m.p.stacked) list = __builtin_amdgcn_readfirstlane((int)at_furthest<NCB, COLS>(row));
        } else {
            const int end = tile0 + ROWS < all ? tile0 + ROWS : all;
            span = at_span_of(x, q, s, (int)((unsigned)tile0 / (unsigned)group), (int)((unsigned)(end - 1) / (unsigned)group));
        }
        walk = at_walk(x.m.p, span.lo0, span.hi1, span.pre1);
        at_part(at_cut(walk, x.m.p), sp, lo, hi);
    }
    const bool none = lo >= hi;
    if (a.n_blocks == 0) hi = lo;
    // with slopes the near tokens come first: far ones weigh less and move no reference (all rows' of a tile would move with
    // each block: 2 x 2048 rows over 16384 tokens, 64 elements, 648 us in the place of 1072, 128 elements 960 in the place of 1406; with positive slopes, that is)
    bool last_first = false;
    if constexpr (MODE == AT_ANY) last_first = x.m.slopes != nullptr;
    auto block = [&](int v) { return MODE == AT_PLAIN ? v : walk.block(last_first ? walk.n - 1 - v : v); };
    const int32_t* pages = a.pages + (int64_t)list * a.pages_stride;
    const uint8_t* kb = (const uint8_t*)a.k + (int64_t)kh * 64 * D;
    const uint8_t* vb = (const uint8_t*)a.v + (int64_t)kh * 64 * D;
    const int64_t step = (int64_t)a.heads * 64 * D;
    uint2 kr[NB][KS], vr[DB][PS];
    // a block that is not there is read as block 0 and hidden
    auto page_of = [&](int v) { return v < hi ? kv_block(pages[block(v)]) : 0; };
    auto there = [&](int p) { return p >= 0 && p < a.n_blocks; };
    auto factors = [&](int p) {
        const float2 f = *(const float2*)(a.scales + ((int64_t)(there(p) ? p : 0) * a.heads + kh) * 2);
        return there(p) ? f : make_float2(1.0f, 1.0f);
    };
    auto load_keys = [&](int page) {
        const uint8_t* base = kb + (there(page) ? page : 0) * step;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint8_t* p = base + M::token(b, n) * D + g * (D / NG);
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
    auto load_values = [&](int page) {
        const uint8_t* base = vb + (there(page) ? page : 0) * step;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            const uint8_t* p = base + (d * COLS + n) * 64 + g * TPL;
#pragma unroll
            for (int t = 0; t < PS; t += 2) {
                const uint4 w = *(const uint4*)(p + 8 * t);
                vr[d][t] = make_uint2(w.x, w.y);
                vr[d][t + 1] = make_uint2(w.z, w.w);
            }
        }
    };

    // the first block is under way before the queries are
    int blk = lo + wk;
    int page = page_of(blk), next = page_of(blk + WK);
    float2 f = make_float2(1.0f, 1.0f);
    if (blk < hi) {
        f = factors(page);
        load_keys(page);
        load_values(page);
    }
    h8 qf[NCB][KS];
    float qc[NCB];
    int pos[NCB];
    load_queries<D, COLS, NCB>(a, q, kh, group, tile0, all, n, g, wide != 0, qf, qc, pos);
    if constexpr (MODE != AT_PLAIN)                          // while the block is under way, where its number did not need them
        if (!(x.m.since || x.m.until || x.m.p.stacked)) find_rows();
    float slope[NCB];
    int anchor[NCB];
    if constexpr (at_slopes(MODE)) load_slopes<MODE, COLS, NCB>(x, kh, group, tile0, all, n, row, slope, anchor);
    bool caps = false, slopes = false;
    float cap_in = 0.0f, cap_out = 0.0f;                     // exp2 of cap_in times a score, and 2 cap in units of the exponents
    if constexpr (MODE == AT_ANY) {
        caps = x.m.cap != 0.0f;
        slopes = x.m.slopes != nullptr;
        if (caps) cap_in = 2.0f / x.m.cap;
        cap_out = 2.0f * 1.44269504088896341f * x.m.cap;
    }
    // tokens [whole_lo, whole_hi) are seen by all rows of the wave: their blocks need no comparisons
    const int last = tile0 + ROWS < all ? tile0 + ROWS : all;
    const int pmin = q.first + (int)((unsigned)tile0 / (unsigned)group), pmax = q.first + (int)((unsigned)(last - 1) / (unsigned)group);
    const int64_t window = a.window > 0 ? a.window : (int64_t)1 << 40;
    const int whole_hi = a.causal ? pmin + 1 : q.len;
    const int whole_lo = pmax - window + 1 > 0 ? (int)(pmax - window + 1) : 0;

    acc o[NCB][DB];
    // weights are exp2(z + lv - m + AT_LIFT); `move`: an exponent above it moves m (any does in a row that has no m yet)
    float m[NCB], l[NCB], move[NCB];
#pragma unroll
    for (int c = 0; c < NCB; ++c) {
        m[c] = 0.0f;
        l[c] = 0.0f;
        move[c] = -3.0e38f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < CREG; ++r) o[c][d][r] = 0.0f;
    }

    float top_f = 0.0f;                                      // the largest value factor so far
    for (; blk < hi; blk += WK) {
        const int after = page_of(blk + 2 * WK);
        const float2 fn = factors(next);
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
        if (blk + WK < hi) load_keys(next);

        const float lv = __builtin_amdgcn_logf(f.y), iv = __builtin_amdgcn_rcpf(f.y);
        const int t0 = block(blk) * 64;
        const bool gone = MODE != AT_PLAIN && !there(page);
        const int len = MODE == AT_PLAIN ? (there(page) ? q.len : t0) : gone ? t0 : max(span.hi1, span.pre1);
        const bool masked = MODE == AT_PLAIN ? t0 + 64 > whole_hi || t0 < whole_lo || t0 + 64 > len
                                             : gone || !(t0 + 64 <= span.pre0 || (t0 >= span.lo1 && t0 + 64 <= span.hi0));
        if (t0 + 64 > len) {                                 // places without a token: their codes may be anything
            const int over = len - t0 - g * TPL;             // the lane's tokens from here on
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int t = 0; t < PS; ++t) {
                    const int x = over - 8 * t, y = x - 4;
                    const uint32_t mx = x >= 4 ? ~0u : x <= 0 ? 0u : (1u << (8 * x & 31)) - 1u;
                    const uint32_t my = y >= 4 ? ~0u : y <= 0 ? 0u : (1u << (8 * y & 31)) - 1u;
                    vr[d][t].x &= mx;
                    vr[d][t].y &= my;
                }
        }
        // exponents of the weights, in place of the scores
        float top[NCB];
#pragma unroll
        for (int c = 0; c < NCB; ++c) {
            const float cz = f.x * qc[c];
            float off = lv - m[c] + AT_LIFT;
            // biases of tokens before all rows rise from token to token; around the rows' own they are made one by one
            const int at = MODE == AT_ANY ? row[c].pos - (t0 + g * TPL) : 0;
            const bool past = MODE == AT_ANY && slopes && t0 + 63 <= span.pos0;
            if (past) off = fmaf(-slope[c], (float)(at - anchor[c]), off);
            if (caps) {
                const float cy = cz * cap_in, oc = off + 0.5f * cap_out;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < CREG; ++r) sc[c][b][r] = capped(sc[c][b][r], cy, cap_out, oc);
            } else {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < CREG; ++r) sc[c][b][r] = fmaf(sc[c][b][r], cz, off);
            }
            if (past) {
#pragma unroll
                for (int t = 1; t < TPL; ++t) sc[c][t / CREG][t % CREG] = fmaf(slope[c], (float)t, sc[c][t / CREG][t % CREG]);
            } else if (slopes) {
#pragma unroll
                for (int t = 0; t < TPL; ++t)
                    sc[c][t / CREG][t % CREG] = fmaf(-slope[c], (float)((at < t ? t - at : at - t) - anchor[c]), sc[c][t / CREG][t % CREG]);
            }
        }
        if (MODE != AT_PLAIN && masked) {
#pragma unroll
            for (int c = 0; c < NCB; ++c) {
                const uint32_t bits = at_bits(row[c], t0 + g * TPL) & (gone ? 0u : ~0u);
#pragma unroll
                for (int t = 0; t < TPL; ++t) sc[c][t / CREG][t % CREG] = at_hidden(sc[c][t / CREG][t % CREG], bits, t);
            }
        }
        if (MODE == AT_PLAIN && masked) {
#pragma unroll
            for (int c = 0; c < NCB; ++c) {
                // the lane's tokens that the row sees
                const int base = t0 + g * TPL;
                const int e = (a.causal && pos[c] < len ? pos[c] : len - 1) - base;
                const int64_t w = pos[c] - window + 1 - base;
                const int seen_lo = w < 0 ? 0 : w > 64 ? 64 : (int)w;
#pragma unroll
                for (int t = 0; t < TPL; ++t)
                    if (t < seen_lo || t > e) sc[c][t / CREG][t % CREG] = -__builtin_inff();
            }
        }
#pragma unroll
        for (int c = 0; c < NCB; ++c) {
            top[c] = sc[c][0][0];
#pragma unroll
            for (int t = 1; t < TPL; ++t) top[c] = fmaxf(top[c], sc[c][t / CREG][t % CREG]);
        }
        bool up = false;
#pragma unroll
        for (int c = 0; c < NCB; ++c) up = up || top[c] > move[c];
        if (__any(up)) {
#pragma unroll
            for (int c = 0; c < NCB; ++c) {
                float x = top[c];
#pragma unroll
                for (int k = COLS; k < 64; k <<= 1) x = fmaxf(x, __shfl_xor(x, k));
                const bool none = move[c] < 0.0f;            // no m yet
                const float by = none ? (x > -1.0e38f ? x - AT_LIFT : 0.0f) : fmaxf(x - AT_LIFT, 0.0f);
                const float shrink = none ? 1.0f : __builtin_amdgcn_exp2f(-by);
                if (x > -1.0e38f) move[c] = AT_LIFT + AT_MOVE;
                m[c] += by;
                l[c] *= shrink;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int r = 0; r < CREG; ++r) o[c][d][r] *= shrink;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < CREG; ++r) sc[c][b][r] -= by;
            }
        }
        h8 pf[NCB][PS];
        const bool low = f.y < top_f * AT_LOW;               // values small beside others': see the factors above
        top_f = fmaxf(top_f, f.y);
#pragma unroll
        for (int c = 0; c < NCB; ++c) {
            float sum = 0.0f, fine = 0.0f;
#pragma unroll
            for (int t = 0; t < PS; ++t)
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const int k = 8 * t + j;
                    const float x = __builtin_amdgcn_exp2f(sc[c][k / CREG][k % CREG]);
                    const float y = __builtin_amdgcn_exp2f(sc[c][(k + 1) / CREG][(k + 1) % CREG]);
                    const h2 p = {(_Float16)x, (_Float16)y};
                    if (HALF) sum = __builtin_amdgcn_fdot2(p, (h2){(_Float16)1.0f, (_Float16)1.0f}, sum, false);
                    if (!HALF || low) fine += x + y;
                    pf[c][t][j] = p[0];
                    pf[c][t][j + 1] = p[1];
                }
            if (!HALF || low) sum = fine;
            // a row that sees nothing of a block takes nothing from a factor that is NaN
            l[c] = masked && sum == 0.0f ? l[c] : fmaf(sum, iv, l[c]);
        }
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int t = 0; t < PS; ++t) {
                const h8 vf = codes8<KT>(vr[d][t]);
#pragma unroll
                for (int c = 0; c < NCB; ++c) o[c][d] = M::run(vf, pf[c][t], o[c][d]);
            }
        if (blk + WK < hi) load_values(next);
        page = next;
        next = after;
        f = fn;
    }
#pragma unroll
    for (int c = 0; c < NCB; ++c)
        if (move[c] < 0.0f) m[c] = AT_NONE;
#pragma unroll
    for (int c = 0; c < NCB; ++c)
#pragma unroll
        for (int k = COLS; k < 64; k <<= 1) l[c] += __shfl_xor(l[c], k);

    {                                                        // one reference for the waves, then their sums in order
        if (g == 0)
#pragma unroll
            for (int c = 0; c < NCB; ++c) ref_sh[wave * COLS * NCB + c * COLS + n] = make_float2(m[c], l[c]);
        __syncthreads();
#pragma unroll
        for (int c = 0; c < NCB; ++c) {
            float2 r[WAVES];
            float top = AT_NONE;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                r[w] = ref_sh[w * COLS * NCB + c * COLS + n];
                top = fmaxf(top, r[w].x);
            }
            const float by = __builtin_amdgcn_exp2f(m[c] - top);
            m[c] = top;
            l[c] = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) l[c] = fmaf(r[w].y, __builtin_amdgcn_exp2f(r[w].x - top), l[c]);
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
#pragma unroll
        for (int w = WAVES / 2; w > 0; w /= 2) {             // halves: the upper waves' sums to the lower ones
            if (wk >= w && wk < 2 * w) put(wk - w);
            __syncthreads();
            if (wk < w) add(wk);
            if (w > 1) __syncthreads();
        }
        if (wk != 0) return;
    }

    store_rows<MODE, D, COLS, NCB>(x, q, s, kh, group, tile0, all, sp, none, n, g, wide != 0, o, m, l);
}

// Many rows: the waves have 32 * NCB rows each and share the blocks.  A block's codes are fetched once for the
// workgroup, a block ahead, and converted into LDS in the order in which lanes read operands (16 bytes a lane).  Half a
// block (32 tokens) at a time, the scores of the next half are made while the weights of the present one are: the matrix
// unit and the vector unit have independent work throughout.  Keys have two buffers and values three, as the products
// with a block's second half run when others convert the next block: one barrier a block.
//
// What the steps gave, 2 x 2048 rows over 16384 tokens of 128 int8 elements, 32 heads on 8 (us): codes from memory to
// registers, 64 rows a wave 2167; converted in LDS 1777, with 32 rows a wave so that two waves fit a SIMD 1462; the order
// of products and vector instructions fenced 1444; conversions spread over the products and LDS slots exchanged against
// bank conflicts 1201; 8 waves to a workgroup 1126; no maximum formed until a sum calls for it 1062; 32-bit arithmetic on
// rows and blocks 1024 (1015 to 1040 from run to run).
template <int MODE, int D, int KT, int NCB, int WAVES, bool HALF>
__global__ void __launch_bounds__(64 * WAVES, D * NCB <= 128 ? 2 : 1) k_kv_attend_tile(AtArgs<MODE> x, int n_tiles, int packed, int wide) {
    const ba_kv_attend_args& a = x.a;
    typedef Mma<32> M;
    typedef M::acc acc;
    constexpr int KS = D / 16, DB = D / 32, T = 64 * WAVES, ROWS = WAVES * 32 * NCB, PC = (4 * D + T - 1) / T;
    __shared__ h8 k_sh[2][8 * D];
    __shared__ h8 v_sh[3][8 * D];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane % 32, g = lane / 32;
    const AtPlace at_wg = at_place(x, ROWS, n_tiles, packed);
    const int tile = at_wg.tile, sp = at_wg.sp, kh = at_wg.kh, s = at_wg.s;
    const int group = a.q_heads / a.heads;
    const AtSeq q = at_rows(x, s);
    const int all = q.rows * group, tile0 = tile * ROWS;
    if (tile < 0 || tile0 >= all) return;
    const int row0 = tile0 + wave * 32 * NCB;
    int lo, hi;
    AtRow row[NCB];
    AtSpan span = {};
    AtWalk walk = {};
    uint4 raw[NCB][KS];
    int list = s;                                            // whose list
    auto find_rows = [&] {
        if constexpr (MODE != AT_PLAIN)
#pragma unroll
            for (int c = 0; c < NCB; ++c) {
                const int r = row0 + c * 32 + n;
                row[c] = at_row(x, q, s, (int)((unsigned)(r < all ? r : all - 1) / (unsigned)group));
            }
    };
    int seen_end = 0;                                        // of the workgroup's rows
    if constexpr (MODE == AT_PLAIN) {
        at_part(at_blocks(a, q, group, tile0, ROWS), sp, lo, hi);
        if (lo >= hi && a.n_splits > 1) return;              // k_kv_join knows which parts there are
    } else {
        int3* span_sh = (int3*)k_sh[1];                      // free until the first block has been converted by all
        int64_t* far_sh = (int64_t*)k_sh[1] + 16;
        if (x.m.since || x.m.until || x.m.p.stacked) find_rows();
        fetch_queries<D, 32, NCB>(a, q, kh, group, row0, all, n, g, wide != 0, raw);
        int3 r;                                              // of all waves
        if (x.m.since || x.m.until || x.m.p.stacked) {
            span = at_span<NCB, 32>(row);
            const int64_t far = x.m.p.stacked ? at_furthest<NCB, 32>(row) : 0;
            if (lane == 0) {
                span_sh[wave] = make_int3(span.lo0, span.hi1, span.pre1);
                far_sh[wave] = far;
            }
            __syncthreads();
            if (x.m.p.stacked) {
                int64_t f = far_sh[0];
#pragma unroll
                for (int w = 1; w < WAVES; ++w) f = far_sh[w] > f ? far_sh[w] : f;
                list = __builtin_amdgcn_readfirstlane((int)f);
            }
            r = span_sh[0];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) r = make_int3(min(r.x, span_sh[w].x), max(r.y, span_sh[w].y), max(r.z, span_sh[w].z));
            r = make_int3(__builtin_amdgcn_readfirstlane(r.x), __builtin_amdgcn_readfirstlane(r.y), __builtin_amdgcn_readfirstlane(r.z));
        } else {
            auto of = [&](int r0, int rows) {
                const int r1 = r0 + rows < all ? r0 + rows : all;
                return at_span_of(x, q, s, (int)((unsigned)(r0 < all ? r0 : all - 1) / (unsigned)group), (int)((unsigned)(r1 - 1) / (unsigned)group));
            };
            span = of(row0, 32 * NCB);
            const AtSpan w = of(tile0, ROWS);
            r = make_int3(w.lo0, w.hi1, w.pre1);
        }
        walk = at_walk(x.m.p, r.x, r.y, r.z);
        seen_end = max(r.y, r.z);
        if (!(x.m.since || x.m.until || x.m.p.stacked)) find_rows();
        at_part(at_cut(walk, x.m.p), sp, lo, hi);
    }
    const bool none = lo >= hi;
    if (a.n_blocks == 0) hi = lo;
    auto block = [&](int v) { return MODE == AT_PLAIN ? v : walk.block(at_slopes(MODE) ? walk.n - 1 - v : v); };   // as above

    h8 qf[NCB][KS];
    float qc[NCB];
    int pos[NCB];
    if constexpr (MODE == AT_PLAIN) load_queries<D, 32, NCB>(a, q, kh, group, row0, all, n, g, wide != 0, qf, qc, pos);
    float slope[NCB];
    int anchor[NCB];
    if constexpr (at_slopes(MODE)) load_slopes<MODE, 32, NCB>(x, kh, group, row0, all, n, row, slope, anchor);
    float cap_in = 0.0f, cap_out = 0.0f;                     // exp2 of cap_in times a score, and 2 cap in units of the exponents
    if constexpr (at_caps(MODE)) {
        cap_in = 2.0f / x.m.cap;
        cap_out = 2.0f * 1.44269504088896341f * x.m.cap;
    }
    // tokens [whole_lo, whole_hi) are seen by all rows of the wave: their blocks need no comparisons
    const int first = row0 < all ? row0 : all - 1, last = row0 + 32 * NCB < all ? row0 + 32 * NCB : all;
    const int pmin = q.first + (int)((unsigned)first / (unsigned)group), pmax = q.first + (int)((unsigned)(last - 1) / (unsigned)group);
    const int64_t window = a.window > 0 ? a.window : (int64_t)1 << 40;
    const int whole_hi = a.causal ? pmin + 1 : q.len;
    const int whole_lo = pmax - window + 1 > 0 ? (int)(pmax - window + 1) : 0;

    acc o[NCB][DB];
    float m[NCB], l[NCB];                                    // weights are exp2(z + lv - m + AT_LIFT)
    bool seen[NCB];                                          // the row has an m
#pragma unroll
    for (int c = 0; c < NCB; ++c) {
        m[c] = 0.0f;
        l[c] = 0.0f;
        seen[c] = false;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[c][d][r] = 0.0f;
    }

    const int32_t* pages = a.pages + (int64_t)list * a.pages_stride;
    const uint8_t* kb = (const uint8_t*)a.k + (int64_t)kh * 64 * D;
    const uint8_t* vb = (const uint8_t*)a.v + (int64_t)kh * 64 * D;
    const int64_t step = (int64_t)a.heads * 64 * D;
    // a block that is not there is read as block 0 and hidden
    auto page_of = [&](int v) { return v < hi ? kv_block(pages[block(v)]) : 0; };
    auto there = [&](int p) { return p >= 0 && p < a.n_blocks; };
    auto factors = [&](int p) {
        const float2 f = *(const float2*)(a.scales + ((int64_t)(there(p) ? p : 0) * a.heads + kh) * 2);
        return there(p) ? f : make_float2(1.0f, 1.0f);
    };
    uint4 kr[PC], vr[PC];                                    // the thread's 16-byte pieces of a block
    auto fetch = [&](int page) {
        const int64_t base = (there(page) ? page : 0) * step;
#pragma unroll
        for (int i = 0; i < PC; ++i) {
            const int u = tid + i * T;
            if (4 * D % T == 0 || u < 4 * D) {
                kr[i] = *(const uint4*)(kb + base + 16 * u);
                vr[i] = *(const uint4*)(vb + base + 16 * u);
            }
        }
    };
    auto hide = [&](int blk, int page) {                     // places without a token: their codes may be anything
        const int len = there(page) ? (MODE == AT_PLAIN ? q.len : seen_end) : blk * 64;
        if (blk * 64 + 64 <= len) return;
#pragma unroll
        for (int i = 0; i < PC; ++i) {
            const int over = len - blk * 64 - 16 * ((tid + i * T) % 4);
            auto keep = [&](uint32_t w, int x) { return w & (x >= 4 ? ~0u : x <= 0 ? 0u : (1u << (8 * x & 31)) - 1u); };
            vr[i].x = keep(vr[i].x, over);
            vr[i].y = keep(vr[i].y, over - 4);
            vr[i].z = keep(vr[i].z, over - 8);
            vr[i].w = keep(vr[i].w, over - 12);
        }
    };
    // LDS places of the thread's pieces.  An operand is 64 slots of 16 bytes, one for each lane; slots are exchanged (by
    // t / 2 and g) so that 8 threads in a row, whose pieces differ in t and g, write to different banks.
    constexpr int SWZ_T = D >= 128 ? 0 : 1, SWZ_G = D == 96 ? 8 : 4;
    int k_at[PC], v_at[PC];
#pragma unroll
    for (int i = 0; i < PC; ++i) {
        const int u = tid + i * T, token = u / (D / 16), e = u % (D / 16) * 16, kg = e / (D / 2), x = (e - kg * (D / 2)) / 8;
        const int b = token >> 4 & 1, kn = (token >> 2 & 3) * 8 + (token >> 5) * 4 + (token & 3);      // M::token turned round
        k_at[i] = (b * KS + x) * 64 + ((kg * 32 + kn) ^ (x / 2 << SWZ_T) ^ (kg * SWZ_G));
        const int d = u / 4, c = u % 4;
        v_at[i] = (d / 32 * 4 + c % 2 * 2) * 64 + ((c / 2 * 32 + d % 32) ^ (c % 2 * 2) ^ (c / 2 * 4));
    }
    const int k_lane = lane ^ (g * SWZ_G), v_lane = lane ^ (g * 4);
    auto convert = [&](int unit, h8* k, h8* v) {             // a quarter of a piece
        const int i = unit / 4;
        if (4 * D % T != 0 && tid + i * T >= 4 * D) return;
        switch (unit % 4) {
            case 0: k[k_at[i]] = codes8<KT>(make_uint2(kr[i].x, kr[i].y)); break;
            case 1: k[k_at[i] + 64] = codes8<KT>(make_uint2(kr[i].z, kr[i].w)); break;
            case 2: v[v_at[i]] = codes8<KT>(make_uint2(vr[i].x, vr[i].y)); break;
            case 3: v[v_at[i] + 64] = codes8<KT>(make_uint2(vr[i].z, vr[i].w)); break;
        }
    };
    // What makes exponents of half b of a block: they are fma(score, cz, off), or of the capped score, and rise by `rise`
    // from token to token.  A lane whose 16 tokens lie on both sides of its row's position takes those after it for tokens
    // before it; settle() puts them right.
    struct Form {
        float cz[NCB], off[NCB], rise[NCB];
    };
    auto form = [&](float2 f, float lv, int blk, int b) {
        Form r;
#pragma unroll
        for (int c = 0; c < NCB; ++c) {
            r.cz[c] = f.x * qc[c];
            r.off[c] = lv - m[c] + AT_LIFT;
            r.rise[c] = 0.0f;
            if constexpr (at_caps(MODE)) {
                r.cz[c] *= cap_in;
                r.off[c] += 0.5f * cap_out;
            }
            if constexpr (at_slopes(MODE)) {
                const int at = row[c].pos - (blk * 64 + 32 * g + 16 * b);
                r.rise[c] = at > 0 ? slope[c] : -slope[c];
                r.off[c] = fmaf(-slope[c], (float)((at > 0 ? at : -at) - anchor[c]), r.off[c]);
            }
        }
        return r;
    };
    // exponents e0 .. e1 of the 16 * NCB that a lane makes from its scores
    auto exponents = [&](acc (&t)[NCB], const Form& r, int e0, int e1) {
#pragma unroll
        for (int e = e0; e < e1; ++e) {
            float y = t[e / 16][e % 16];
            if constexpr (at_caps(MODE)) y = capped(y, r.cz[e / 16], cap_out, r.off[e / 16]);
            else y = fmaf(y, r.cz[e / 16], r.off[e / 16]);
            if constexpr (at_slopes(MODE)) y = fmaf(r.rise[e / 16], (float)(e % 16), y);
            t[e / 16][e % 16] = y;
        }
    };
    // moves the reference of rows: m, l and the sums, and the exponents at hand
    auto move_by = [&](acc (&t)[NCB], int c, float by) {
        const float shrink = __builtin_amdgcn_exp2f(-by);
        m[c] += by;
        l[c] *= shrink;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[c][d][r] *= shrink;
#pragma unroll
        for (int r = 0; r < 16; ++r) t[c][r] -= by;
    };
    auto largest = [&](const acc (&t)[NCB], int c) {
        float x = t[c][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) x = fmaxf(x, t[c][r]);
        return fmaxf(x, __shfl_xor(x, 32));
    };
    // what most blocks do not need: tokens hidden from rows, and the first reference of a row
    bool unset = true;                                       // a row of the wave has none
    float top_f = 0.0f;                                      // the largest value factor so far
    auto settle = [&](acc (&t)[NCB], int blk, int page, int b) {
        const int t0 = blk * 64, len = there(page) ? q.len : t0;
        const bool gone = MODE != AT_PLAIN && !there(page);
        const bool masked = MODE == AT_PLAIN ? t0 + 64 > whole_hi || t0 < whole_lo || t0 + 64 > len
                                             : gone || !(t0 + 64 <= span.pre0 || (t0 >= span.lo1 && t0 + 64 <= span.hi0));
        const bool both = at_slopes(MODE) && t0 + 64 > span.pos0 && t0 <= span.pos1;       // sides of a row's position
        if (!masked && !unset && !both) return;
        bool none = false;
#pragma unroll
        for (int c = 0; c < NCB; ++c) {
            if constexpr (at_slopes(MODE))
                if (both) {
                    const int at = row[c].pos - (t0 + 32 * g + 16 * b), from = at > 0 ? at : 16;
#pragma unroll
                    for (int r = 2; r < 16; ++r) t[c][r] = fmaf(-2.0f * slope[c], (float)max(r - from, 0), t[c][r]);
                }
            if constexpr (MODE != AT_PLAIN)
                if (masked) {
                    const uint32_t bits = at_bits(row[c], t0 + 32 * g + 16 * b) & (gone ? 0u : ~0u);
#pragma unroll
                    for (int r = 0; r < 16; ++r) t[c][r] = at_hidden(t[c][r], bits, r);
                }
            if (MODE == AT_PLAIN && masked) {                                    // the lane's tokens that the row sees
                const int base = t0 + 32 * g + 16 * b;
                const int e = (a.causal && pos[c] < len ? pos[c] : len - 1) - base;
                const int64_t w = pos[c] - window + 1 - base;
                const int seen_lo = w < 0 ? 0 : w > 64 ? 64 : (int)w;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (r < seen_lo || r > e) t[c][r] = -__builtin_inff();
            }
            if (unset) {
                const float x = largest(t, c);
                const bool sets = !seen[c] && x > -1.0e38f;
                if (sets) {                                  // its sums are zeros
                    m[c] = x - AT_LIFT;
#pragma unroll
                    for (int r = 0; r < 16; ++r) t[c][r] -= m[c];
                    seen[c] = true;
                }
                none = none || !seen[c];
            }
        }
        if (unset) unset = __any(none);
    };
    // One half block: the scores of another half (keys k, at half kb2 of their block; factors fn) into tn, the weights and
    // products of the present one (exponents t, values v at half vb2, factors f).  The matrix unit takes a product every
    // 32 clocks; vector instructions stand between them in the order that the fences keep.  Operands are read AHEAD
    // products ahead, with `carry` through the end of the half into the second half of k, the next one's keys.
    constexpr int AHEAD = D == 32 ? 2 : 4, READS = KS + 2 * DB, STEPS = 2 * DB * NCB;
    h8 ring[AHEAD];
    auto key = [&](const h8* k, int b, int x) { return k[(b * KS + x) * 64 + (k_lane ^ (x / 2 << SWZ_T))]; };
    auto half = [&](acc (&t)[NCB], acc (&tn)[NCB], const h8* k, int kb2, const h8* v, int vb2, float2 f, float2 fn, int blkn, auto carry, auto extra) {
        constexpr int PAIRS = 8 * NCB, EL = 16 * NCB;
        auto read = [&](int i) {
            if (i < KS) ring[i % AHEAD] = key(k, kb2, i);
            else if (i < READS) ring[i % AHEAD] = v[((i - KS) % DB * 4 + 2 * vb2 + (i - KS) / DB) * 64 + (v_lane ^ (2 * vb2))];
            else if constexpr (decltype(carry)::value) ring[i % AHEAD] = key(k, 1, i - READS);
        };
        h8 pf[NCB][2];
        float sum[NCB];
        const bool low = HALF && f.y < top_f * AT_LOW;       // values small beside others': see the factors above
        top_f = fmaxf(top_f, f.y);
        auto weigh = [&](int i0, int i1) {
#pragma unroll
            for (int i = i0; i < i1; ++i) {
                const int c = i % NCB, j = i / NCB * 2;
                const float y = __builtin_amdgcn_exp2f(t[c][j]), z = __builtin_amdgcn_exp2f(t[c][j + 1]);
                const h2 p = {(_Float16)y, (_Float16)z};
                if (HALF) sum[c] = __builtin_amdgcn_fdot2(p, (h2){(_Float16)1.0f, (_Float16)1.0f}, sum[c], false);
                else sum[c] += y + z;
                pf[c][j / 8][j % 8] = p[0];
                pf[c][j / 8][j % 8 + 1] = p[1];
            }
        };
#pragma unroll
        for (int c = 0; c < NCB; ++c) {
            sum[c] = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; ++r) tn[c][r] = 0.0f;
        }
        // the wave that is at its exponentials goes first: the other one's products fill the matrix unit meanwhile
        // (2 x 2048 rows over 16384 tokens, 64 elements: 580 -> 564 us)
        __builtin_amdgcn_s_setprio(1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < KS; ++x) {
#pragma unroll
            for (int c = 0; c < NCB; ++c) {                  // a product's 32 clocks are the next pairs' time
                const int i = x * NCB + c;
                tn[c] = M::run(ring[x % AHEAD], qf[c][x], tn[c]);
                if (c == NCB - 1) read(x + AHEAD);
                weigh(i * PAIRS / (KS * NCB), (i + 1) * PAIRS / (KS * NCB));
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_s_setprio(0);
        // weights that fp16 could not hold show in their sum: no maximum is formed until then
        bool rare = low, big = false;
#pragma unroll
        for (int c = 0; c < NCB; ++c) big = big || sum[c] > AT_MOST;
        rare = rare || big;
        if (__any(rare)) {
            if (__any(big)) {
#pragma unroll
                for (int c = 0; c < NCB; ++c) {
                    const float x = largest(t, c);
                    move_by(t, c, x > AT_LIFT ? x - AT_LIFT : 0.0f);
                    sum[c] = 0.0f;
                }
                weigh(0, PAIRS);
            }
            if (HALF && low)
#pragma unroll
                for (int c = 0; c < NCB; ++c) {
                    sum[c] = 0.0f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum[c] += __builtin_amdgcn_exp2f(t[c][r]);
                }
        }
        const float iv = __builtin_amdgcn_rcpf(f.y), lv = __builtin_amdgcn_logf(fn.y);
#pragma unroll
        for (int c = 0; c < NCB; ++c)                        // a row that sees nothing of a block takes nothing from a factor that is NaN
            l[c] = sum[c] == 0.0f ? l[c] : fmaf(sum[c], iv, l[c]);
        const Form next = form(fn, lv, blkn, kb2);
#pragma unroll
        for (int x = 0; x < 2 * DB; ++x) {
#pragma unroll
            for (int c = 0; c < NCB; ++c) {
                const int i = x * NCB + c;
                o[c][x % DB] = M::run(ring[(KS + x) % AHEAD], pf[c][x / DB], o[c][x % DB]);
                if (c == NCB - 1) read(KS + x + AHEAD);
                extra(i);
                if (i > 0) exponents(tn, next, (i - 1) * EL / (STEPS - 1), i * EL / (STEPS - 1));
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    auto preload = [&](const h8* k, int b) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) ring[i] = key(k, b, i);
    };
    // LDS written before is visible after; global loads may be in flight across it
    auto meet = [&] {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    if (lo < hi) {
        int page = page_of(lo), next = page_of(lo + 1);
        float2 f = factors(page);
        acc t0[NCB], t1[NCB];
        fetch(page);
        if constexpr (MODE != AT_PLAIN) shape_queries<D, 32, NCB>(a, raw, qf, qc);
        hide(block(lo), page);
#pragma unroll
        for (int i = 0; i < 4 * PC; ++i) convert(i, k_sh[0], v_sh[0]);
        fetch(next);
        meet();
        {                                                    // scores of the first half
#pragma unroll
            for (int c = 0; c < NCB; ++c) {
#pragma unroll
                for (int r = 0; r < 16; ++r) t0[c][r] = 0.0f;
#pragma unroll
                for (int x = 0; x < KS; ++x) t0[c] = M::run(key(k_sh[0], 0, x), qf[c][x], t0[c]);
            }
            exponents(t0, form(f, __builtin_amdgcn_logf(f.y), block(lo), 0), 0, 16 * NCB);
        }
        settle(t0, block(lo), page, 0);
        preload(k_sh[0], 1);
        int kc = 0, vc = 0;                                  // buffers of the present block
        for (int blk = lo; blk < hi; ++blk) {
            // after the last block the next one is block 0, converted into free buffers and not used
            const int after = page_of(blk + 2), vn = vc == 2 ? 0 : vc + 1;
            const float2 fn = factors(next);
            hide(block(blk + 1), next);
            half(t0, t1, k_sh[kc], 1, v_sh[vc], 0, f, f, block(blk), std::false_type(), [&](int x) {
#pragma unroll
                for (int i = x * 4 * PC / STEPS; i < (x + 1) * 4 * PC / STEPS; ++i) convert(i, k_sh[kc ^ 1], v_sh[vn]);
                if (x == STEPS - 1) fetch(after);            // the registers that were converted are free
            });
            settle(t1, block(blk), page, 1);
            meet();
            preload(k_sh[kc ^ 1], 0);
            half(t1, t0, k_sh[kc ^ 1], 0, v_sh[vc], 1, f, fn, block(blk + 1), std::true_type(), [](int) {});
            if (blk + 1 < hi) settle(t0, block(blk + 1), next, 0);
            kc ^= 1;
            vc = vn;
            page = next;
            next = after;
            f = fn;
        }
    }
#pragma unroll
    for (int c = 0; c < NCB; ++c) {
        if (!seen[c]) m[c] = AT_NONE;
        l[c] += __shfl_xor(l[c], 32);
    }
    store_rows<MODE, D, 32, NCB>(x, q, s, kh, group, row0, all, sp, none, n, g, wide != 0, o, m, l);
}

// The parts of each row joined: a thread takes 4 elements, `lanes` groups of threads the parts in turn.
template <int MODE>
__global__ void __launch_bounds__(AT_T) k_kv_join(AtArgs<MODE> x, int tile_rows, int lanes, int wide) {
    const ba_kv_attend_args& a = x.a;
    __shared__ f4 sum_sh[AT_T];
    __shared__ float den_sh[AT_T];
    const int quads = a.dim / 4, unit = threadIdx.x / quads, d = threadIdx.x % quads * 4;
    const int per_wg = AT_T / quads / lanes;                 // rows of a workgroup
    const unsigned rh = blockIdx.x * (unsigned)per_wg + unit / lanes;
    const int lane = unit % lanes;
    const int64_t row = rh / (unsigned)a.q_heads;
    const int head = (int)(rh - (unsigned)row * a.q_heads);
    const bool mine = unit / lanes < per_wg && row < a.n_rows;
    f4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    float den = 0.0f, top = AT_NONE;
    bool covered = false;
    int n = 0;                                               // parts of the row
    float shift = 0.0f;
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
        if constexpr (MODE != AT_PLAIN) {                    // parts without blocks say so
            if (covered) {
                n = a.n_splits;
                for (int p = lane; p < n; p += lanes) top = fmaxf(top, part_ref(a, row, head, p)->x);
                if (a.lse && d == 0 && lane == 0 && x.m.slopes) shift = lse_shift(x, at_row(x, q, s, i), head);
            }
        } else if (covered) {
            const int r = (int)i * group + head % group;
            const AtBlocks b = at_blocks(a, q, group, r / tile_rows * tile_rows, tile_rows);
            n = (b.hi - b.lo + b.per - 1) / b.per;
            for (int p = lane; p < n; p += lanes) top = fmaxf(top, part_ref(a, row, head, p)->x);
        }
    }
    // one reference for the row
    den_sh[threadIdx.x] = top;
    __syncthreads();
    if (mine)                                                // threads left over have no group of their own
        for (int k = 0; k < lanes; ++k) top = fmaxf(top, den_sh[threadIdx.x + (k - lane) * quads]);
    __syncthreads();
    for (int p = lane; p < n; p += lanes) {
        const float2 f = *part_ref(a, row, head, p);
        if (MODE != AT_PLAIN && f.x == AT_NONE && f.y == 0.0f) continue;     // (a row whose scores are NaN has no reference either)
        const float by = __builtin_amdgcn_exp2f(f.x - top);
        const f4 v = *(const f4*)(part_sum(a, row, head, p) + d);
        den = fmaf(f.y, by, den);
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] = fmaf(v[k], by, sum[k]);
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
    if (a.lse && d == 0) {
        const float lse = den == 0.0f ? -__builtin_inff() : 0.693147180559945309f * (top - AT_LIFT + __builtin_amdgcn_logf(den));
        a.lse[row * a.q_heads + head] = MODE == AT_PLAIN ? lse : lse - shift;
    }
}

// The kernel for a call by the rows that share a cache head: up to 16 in 16 columns and up to 32 in 32 with the waves
// splitting the blocks; more in workgroups of 128 rows or, from 129 on, of 256 that share the converted blocks (128 where
// heads of 256 leave a wave registers for 32 rows only).  256 rows are 4 waves of 64 rows up to 64 elements a head, and 8
// waves of 32 above: then two waves fit a SIMD (2 x 2048 rows over 16384 tokens, before the last steps of the kernel: 64
// elements 615 us against 690 with 8 waves, 128 elements 1077 us against 1375 with 4).  `fit`: workgroups that a CU holds.
struct AtShape { int cols, ncb, waves, rows, fit; };
static inline AtShape at_tile(int rows, int dim) {
    if (rows == 16) return {16, 0, 4, 16, dim <= 64 ? 4 : dim <= 128 ? 2 : 1};
    if (rows == 32) return {32, 0, 4, 32, dim <= 128 ? 2 : 1};
    if (rows == 128 || dim > 128) return {32, 1, 4, 128, dim <= 64 ? 3 : dim <= 128 ? 2 : 1};
    if (dim <= 64) return {32, 2, 4, 256, 2};
    return {32, 1, 8, 256, 1};
}
static inline AtShape at_shape(int64_t rows, int dim) { return at_tile(rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 128 ? 128 : 256, dim); }

#define AT_WINDOW ((int64_t)1 << 40)      // wider ones are no narrower to any position, and sums with them pass 64 bits
static inline int64_t at_window(int64_t window) { return window < AT_WINDOW ? window : AT_WINDOW; }

// The checks and sizes of every attention call (ba_kv_attend.hip).
struct AtGrid { unsigned nb; int tiles, packed; };
struct AtJoin { int lanes; unsigned nb; };
int attend_check(const ba_kv_attend_args& a, bool& nothing);
int attend_grid(const ba_kv_attend_args& a, int64_t rows, int64_t n_seqs, int parts, const AtShape& v, AtGrid& g);
int attend_join(const ba_kv_attend_args& a, AtJoin& j);
int attend_wide(const ba_kv_attend_args& a);

// Launches of the kernels for few rows and of those for tiles; each mode's are made in a source of their own.
template <int MODE, int D, int KT, bool HALF>
static void launch_few(const AtArgs<MODE>& x, const AtShape& v, const AtGrid& g, int wide, hipStream_t st) {
    const dim3 grid(g.nb), block(64 * v.waves);
    if (v.cols == 16) hipLaunchKernelGGL((k_kv_attend<MODE, D, KT, 16, HALF>), grid, block, 0, st, x, g.tiles, g.packed, wide);
    else hipLaunchKernelGGL((k_kv_attend<MODE, D, KT, 32, HALF>), grid, block, 0, st, x, g.tiles, g.packed, wide);
}

template <int MODE, int D, int KT, bool HALF>
static void launch_tiles(const AtArgs<MODE>& x, const AtShape& v, const AtGrid& g, int wide, hipStream_t st) {
    const dim3 grid(g.nb), block(64 * v.waves);
    if (v.rows == 128) hipLaunchKernelGGL((k_kv_attend_tile<MODE, D, KT, 1, 4, HALF>), grid, block, 0, st, x, g.tiles, g.packed, wide);
    else if constexpr (D <= 64) hipLaunchKernelGGL((k_kv_attend_tile<MODE, D, KT, 2, 4, HALF>), grid, block, 0, st, x, g.tiles, g.packed, wide);
    else if constexpr (D <= 128) hipLaunchKernelGGL((k_kv_attend_tile<MODE, D, KT, 1, 8, HALF>), grid, block, 0, st, x, g.tiles, g.packed, wide);
}

#define AT_LAUNCH(NAME)                                                                                                   \
    template <int MODE, int D>                                                                                            \
    static int NAME##_of(const AtArgs<MODE>& x, const AtShape& v, const AtGrid& g, int wide, hipStream_t st) {            \
        const bool half = x.a.dtype == BA_F16;                                                                            \
        if (x.a.bits == BA_FP8) half ? NAME<MODE, D, BA_FP8, true>(x, v, g, wide, st) : NAME<MODE, D, BA_FP8, false>(x, v, g, wide, st);   \
        else half ? NAME<MODE, D, BA_INT8, true>(x, v, g, wide, st) : NAME<MODE, D, BA_INT8, false>(x, v, g, wide, st);   \
        BA_LAUNCHED();                                                                                                    \
        return BA_OK;                                                                                                     \
    }                                                                                                                     \
    template <int MODE>                                                                                                   \
    int NAME(const AtArgs<MODE>& x, const AtShape& v, const AtGrid& g, int wide, hipStream_t st) {                        \
        switch (x.a.dim) {                                                                                                \
            case 32: return NAME##_of<MODE, 32>(x, v, g, wide, st);                                                       \
            case 64: return NAME##_of<MODE, 64>(x, v, g, wide, st);                                                       \
            case 96: return NAME##_of<MODE, 96>(x, v, g, wide, st);                                                       \
            case 128: return NAME##_of<MODE, 128>(x, v, g, wide, st);                                                     \
            case 256: return NAME##_of<MODE, 256>(x, v, g, wide, st);                                                     \
        }                                                                                                                 \
        return BA_ERR_UNSUPPORTED;                                                                                        \
    }
AT_LAUNCH(launch_few)
AT_LAUNCH(launch_tiles)
#undef AT_LAUNCH

}  // namespace ba
