// Attention over the 8-bit cache with formed scores, masks by row and sequences that begin alike.
//
//   z_j = scale q.k_j;  with a cap: cap tanh(z_j / cap);  with slopes: less slope |p - j|
//   o = sum_j e^z_j v_j / sum_j e^z_j  over the tokens j that a row sees:
//   j < prefix of its sequence, or since <= j < until of the row, causal and in the window
//
// The kernels are those of ba_kv_attend.h.  What a row sees is two intervals there (AtRow), and a workgroup walks over the
// blocks that any of its rows sees (AtWalk): a window behind a prefix, or a document in a long prompt, costs its own blocks.
//
// shared: the first so many blocks of all lists that have tokens there are the same.  One launch takes the rows of all sequences
// over these blocks as if they were one sequence's (AtPart.stacked), another, or the rest of the same, each sequence's own
// blocks, and both leave partial sums for one join: the shared tokens are read, and converted, once for up to 256 rows instead
// of once for each sequence.
//
// Measured (heads of 128 int8, 32 on 8, unless said otherwise):
//   memory   48 sequences of up to 8192 tokens, a token each, slopes: 91 us (4.6 TB/s) + join 5, as without slopes; 16 of 65000
//            that see 64 + 4096 tokens, e4m3: 32 us (4.3 TB/s) + 5
//   issue    2 x 2048 rows over 16384 tokens: 1030 us with masks, 960 with slopes (far weights vanish, and power with them), 1200
//            capped (vector units busy 64% of the time, 27 of it two transcendentals a score; the matrix unit 35%, 21 of it beside them;
//            22% of the time neither: barriers, LDS and what waits for what in a wave), 1180 both
//   latency  8192 tokens of documents of 50 to 2000: 149 us, where their products would take 65 (documents of 64, one block a tile:
//            54, in four turns of two tiles a CU: that is what a tile takes to begin and end)
//   shared   64 tokens over 16384 shared and 1 to 512 of their own: 45 + 6 us (41 + 16 + 6 as two launches); read by each, 460
//   16 heads of 64, e4m3: 6144 rows of frames over 12288 tokens 290 us (0.83 PFLOP/s), 4608 rows of six frames over 16128 391 us
#include <math.h>

#include "ba_kv_attend.h"

namespace ba {

#define SC_MIN_BLOCKS 4      // blocks of a part of a tile at least

#define AT_ELSEWHERE(NAME, MODE) extern template int NAME<MODE>(const AtArgs<MODE>&, const AtShape&, const AtGrid&, int, hipStream_t);
AT_ELSEWHERE(launch_few, AT_ANY)
AT_ELSEWHERE(launch_tiles, AT_MASKS)
AT_ELSEWHERE(launch_tiles, AT_SLOPES)
AT_ELSEWHERE(launch_tiles, AT_CAPPED)
AT_ELSEWHERE(launch_tiles, AT_BOTH)
#undef AT_ELSEWHERE

static int launch_formed(const ba_kv_attend_args& a, const AtMore& m, const AtShape& v, const AtGrid& g, int wide, hipStream_t st) {
    if (!v.ncb) return launch_few(AtArgs<AT_ANY>{a, m, {}}, v, g, wide, st);
    if (m.cap != 0.0f) return m.slopes ? launch_tiles(AtArgs<AT_BOTH>{a, m}, v, g, wide, st) : launch_tiles(AtArgs<AT_CAPPED>{a, m}, v, g, wide, st);
    return m.slopes ? launch_tiles(AtArgs<AT_SLOPES>{a, m}, v, g, wide, st) : launch_tiles(AtArgs<AT_MASKS>{a, m}, v, g, wide, st);
}

static bool joint_shape(const AtShape& own, const AtShape& common, double wgs) {
    return !own.ncb && !common.ncb && (own.rows >= common.rows || wgs <= 1024.0);
}

// The launches of a call: of the sequences' own blocks, of the shared ones, and the join's.
struct ScoredShape {
    AtShape v, w;
    AtGrid g, h;
    AtJoin j;
    bool joint;
};

// a: the call's, with all of its parts.  Errors are those of sizes and of the workspace.
static int scored_shape(const ba_kv_scored_args& s, const ba_kv_attend_args& a, ScoredShape& r) {
    const int group = a.q_heads / a.heads;
    const int64_t rows = a.max_rows * group, all = a.n_rows * group;
    r.v = s.tile ? at_tile(s.tile, a.dim) : at_shape(rows, a.dim);
    r.w = s.shared_tile ? at_tile(s.shared_tile, a.dim) : at_shape(all, a.dim);
    // both in one launch, where that takes the sequences' own no larger tile or they are few (2048 workgroups of tokens over 164
    // tokens in tiles of 16 rows: 50 us, 63 in tiles of 32)
    r.joint = s.shared && joint_shape(r.v, r.w, (double)a.n_seqs * a.heads);
    if (r.joint) r.v = r.w = r.v.rows > r.w.rows ? r.v : r.w;
    int rc = attend_grid(a, rows, a.n_seqs, s.a.n_splits, r.v, r.g);
    if (rc == BA_OK && s.shared) rc = attend_grid(a, all, 1, s.shared_parts, r.w, r.h);
    if (rc == BA_OK) rc = attend_join(a, r.j);
    if (rc != BA_OK) return rc;
    BA_REQUIRE(!r.joint || r.g.nb < (1u << 23) - r.h.nb, "attention: too many tiles for a call");
    return BA_OK;
}

static int attend_scored(const ba_kv_scored_args& s, hipStream_t st) {
    ba_kv_attend_args a = s.a;
    a.window = at_window(a.window);
    a.n_splits = s.a.n_splits + s.shared_parts;
    ScoredShape shape;
    int rc = scored_shape(s, a, shape);
    if (rc != BA_OK) return rc;
    const AtShape &v = shape.v, &w = shape.w;
    const AtGrid &g = shape.g, &h = shape.h;
    const AtJoin& j = shape.j;
    const bool joint = shape.joint;
    auto least = [](const AtShape& x) { return x.ncb ? SC_MIN_BLOCKS : AT_MIN_BLOCKS; };
    const unsigned at_once = BA_N_XCD * (unsigned)g.tiles;
    // unequal: what a tile sees grows with its place by a quarter of the longest's at least (2048 rows over 16384 tokens 1219 us, 1236 dealt out)
    const bool unequal = v.ncb && ((a.causal && !s.since) || s.until) && 4 * a.max_rows >= 64 * (int64_t)a.n_pages;
    const int mix = !unequal ? -1 : g.nb % at_once == 0 ? (int)(g.nb / at_once) : 0;
    const int wide = attend_wide(a);
    AtMore m = {s.slopes, s.prefix, s.since, s.until, s.cap, mix, {s.shared, a.n_pages, s.shared_parts, s.a.n_splits, least(v), 0, g.tiles, g.packed, 0, g.nb}};
    if (s.shared) {
        const AtMore common = {s.slopes, s.prefix, s.since, s.until, s.cap, -1, {0, s.shared, 0, s.shared_parts, least(w), 1, h.tiles, h.packed, 0, h.nb}};
        if (joint) {
            m.p.first = h.nb;
            rc = launch_few(AtArgs<AT_ANY>{a, common, m.p}, v, {h.nb + g.nb, 0, 0}, wide, st);
        } else {
            rc = launch_formed(a, common, w, h, wide, st);
        }
        if (rc != BA_OK) return rc;
    }
    if (!joint) rc = launch_formed(a, m, v, g, wide, st);
    if (rc != BA_OK || a.n_splits == 1) return rc;
    hipLaunchKernelGGL(k_kv_join<AT_ANY>, dim3(j.nb), dim3(AT_T), 0, st, AtArgs<AT_ANY>{a, m, {}}, v.rows, j.lanes, wide);
    BA_LAUNCHED();
    return BA_OK;
}

// What a launch is expected to take (us), which shapes and parts are chosen by.  A CU holds `fit` workgroups at a time and takes
// its share of all of them in turns of so many; a workgroup's time is its blocks' and that of SC_START more to begin and end
// with, and a block's (us, by how many workgroups share the CU) what calls of 2 x 2048 rows over 16384 tokens, of 6144 over
// 12288, of documents of 64 tokens and of 64 to 512 rows over 4096 to 32000 took.  Rows of one tile of 16 or 32 are bound by
// memory: the bytes of the blocks at 4.8 TB/s, or the blocks of a wave in series.  Partial sums add a launch, and their bytes
// go through the caches.  `share`: that of the bound on blocks that tiles see on the average, where each CU has several.
#define SC_START 5

struct Guess {
    AtShape v;
    int parts;
    double us;
};

static double launch_us(const AtShape& v, int dim, double base, int64_t blocks, int parts, double share) {
    const double per = (double)((blocks + parts - 1) / parts);
    static const double rows32[5][2] = {{0.33, 0.2}, {0.42, 0.28}, {0.52, 0.35}, {0.6, 0.41}, {1.2, 0.0}};
    static const double rows128[5][3] = {{0.7, 0.5, 0.43}, {1.2, 0.66, 0.6}, {1.5, 0.93, 0.0}, {1.7, 1.09, 0.0}, {2.45, 0.0, 0.0}};
    static const double rows256[4][2] = {{1.4, 0.94}, {1.6, 1.13}, {1.78, 0.0}, {2.03, 0.0}};
    const int d = dim <= 96 ? dim / 32 - 1 : dim == 128 ? 3 : 4;
    const double* block = v.rows == 256 ? rows256[d] : v.rows == 128 ? rows128[d] : rows32[d];
    const double each = ceil(base * parts / 256.0), full = floor(each / v.fit);
    const int rest = (int)(each - full * v.fit);
    return 4.0 + ((each >= 2.0 ? per * share : per) + (v.rows == 256 ? SC_START + 2 : SC_START)) * (full * v.fit * block[v.fit - 1] + (rest ? rest * block[rest - 1] : 0.0));
}

static double few_us(int dim, double base, int64_t blocks, int parts) {
    const double bytes = base * blocks * 128.0 * dim / 4.8e6, chain = (double)(((blocks + parts - 1) / parts + 3) / 4);
    return 6.0 + (bytes > chain ? bytes : chain);
}

// The best shape and number of parts for the rows of n_seqs sequences that may see `blocks` blocks each; join: time that a part
// more of all rows costs; joined: there is a join anyway; brief: rows see a short part of their lists; beside: another launch
// of the call, which few rows take in where the CUs have room for both.
static Guess guess(int64_t rows, int64_t n_seqs, int heads, int dim, int64_t blocks, double join, bool joined, bool brief, double share,
                   const Guess* beside = nullptr, double beside_wgs = 0.0) {
    auto with = [&](const AtShape& v, double wgs, double us) {
        if (!beside) return us;
        if (!joint_shape(beside->v, v, beside_wgs)) return us + beside->us + 4.0;
        return us + (wgs > 256.0 * (v.fit - 1) || beside->us > us ? beside->us : 2.0);
    };
    Guess best = {at_shape(rows, dim), 1, 0.0};
    if (blocks < 1) blocks = 1;
    // (partial sums of large tiles end their workgroups later than the model's blocks say: 64 rows over 16000 tokens, heads of 64,
    // 40 us in 32 parts of 128 rows, 32 in 8 of 32)
    auto parted = [&](int p, bool large) { return p > 1 || joined ? join * p + (large ? 14.0 : 6.0) + (joined ? 0.0 : 4.0) : 0.0; };
    if (!best.v.ncb) {                                       // one and a half workgroups per CU, two parts for unequal lengths
        // (a list of less than two parts stays whole: 8 x 5 rows over 1100 tokens 10.9 us, 13.9 in two)
        const int64_t base = n_seqs * heads, most = blocks / AT_MIN_BLOCKS;
        int64_t n = (384 + base - 1) / base;
        n = n < 2 && !joined ? 2 : n;
        n = n < most ? n : most;
        best.parts = (int)(n < 1 ? 1 : n);
        best.us = with(best.v, (double)base * best.parts, few_us(dim, (double)base, blocks, best.parts) + parted(best.parts, false));
        return best;
    }
    // documents packed into a prompt are short beside it: small tiles, whole (8192 tokens of documents of 50 to 2000, 32 heads of 128
    // on 8, fp16: 143 us, 146 with tiles of 256 rows, 263 in two parts; 16 heads of 64, bf16: 74, 102)
    if (brief) return {at_tile(128, dim), 1, launch_us(at_tile(128, dim), dim, (double)n_seqs * heads * ((rows + 127) / 128), blocks, 1, 1.0)};
    static const int some[] = {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 16, 20, 24, 32, 40, 48, 64};
    best.us = 1.0e30;
    for (const int tile : {32, 128, 256}) {
        if (tile == 256 && (dim > 128 || rows <= 128)) break;
        const AtShape v = at_tile(tile, dim);
        const int least = v.ncb ? SC_MIN_BLOCKS : AT_MIN_BLOCKS;
        const double base = (double)n_seqs * heads * ((rows + tile - 1) / tile);
        for (const int p : some) {
            if (p > 1 && (int64_t)p * least > blocks) break;
            const double us = with(v, base * p, launch_us(v, dim, base, blocks, p, share) + parted(p, v.ncb != 0));
            if (us < best.us) best = {v, p, us};
        }
    }
    return best;
}

// What a plan may ask for: launches and a join that can be made, and less room for partial sums than 8 GB, 3% of the chip's
// (64 x 2048 rows of 32 heads of 128 over shared blocks take 4.4 in two parts).
#define SC_ROOM ((int64_t)8 << 30)

static bool can_be_made(const ba_kv_scored_args& s) {
    ba_kv_attend_args a = s.a;
    a.n_splits = s.a.n_splits + s.shared_parts;
    a.workspace = (void*)16;                                 // there will be one
    a.workspace_bytes = (int64_t)1 << 62;
    ScoredShape r;
    const bool ok = scored_shape(s, a, r) == BA_OK && ba_kv_attend_workspace_bytes(a.n_rows, a.q_heads, a.dim, a.n_splits) <= SC_ROOM;
    clear_error();
    return ok;
}

}  // namespace ba

using namespace ba;

extern "C" void ba_kv_scored_plan(ba_kv_scored_args* args) {
    ba_kv_attend_args& a = args->a;
    clear_error();
    a.n_splits = 1;
    args->shared_parts = args->shared > 0 ? 1 : 0;
    args->tile = args->shared_tile = 0;
    if (a.n_seqs < 1 || a.heads < 1 || a.q_heads < a.heads || a.max_rows < 1 || a.n_rows < 1 || args->shared < 0 || args->shared > a.n_pages) return;
    const int group = a.q_heads / a.heads;
    const int64_t rows = a.max_rows * group, all = a.n_rows * group;
    const double join = 8.0 * a.n_rows * a.q_heads * (a.dim + 2) / 9.0e6;        // mostly in the caches
    // rows with a first token of their own are taken for those of short documents where they are half of their list (4096 of 8192,
    // 32 heads on 8: 98 us, 104 planned as without; of one long document 449 and 409), or as many as fill the chip whatever they
    // see (2048 in a table of 131072: 47 and 53; 16 heads of 64, 4096: 52 and 65; of one document of 32768: 696 and 587).  Fewer may
    // as well be the end of a long one: 16 rows over 65536 tokens 1666 us and 49, 256 over 8192 202 and 71 (of short documents 29.5 and 26)
    const bool brief = args->since && (2 * a.max_rows >= 64 * (int64_t)a.n_pages || (double)a.n_seqs * a.heads * (rows / 128) >= 512.0);
    int64_t blocks = a.n_pages;
    if (a.window > 0 && a.window < AT_WINDOW && !args->prefix) {                     // what a tile's rows can see
        const int64_t at_once = 256 / group < a.max_rows ? 256 / group + 1 : a.max_rows, seen = (a.window + at_once + 62) / 64 + 1;
        blocks = seen < blocks ? seen : blocks;
    }
    // causal tiles of a prompt see half of what is new on the average
    const double fresh = (double)a.max_rows / (64.0 * (blocks < 1 ? 1 : blocks)), share = a.causal ? 1.0 - 0.5 * (fresh < 1.0 ? fresh : 1.0) : 1.0;
    const Guess own = guess(rows, a.n_seqs, a.heads, a.dim, blocks, join, false, brief, share);
    a.n_splits = own.parts;
    args->tile = own.v.rows;
    if (args->shared > 0) {
        const int64_t rest = a.n_pages - args->shared;
        const Guess left = guess(rows, a.n_seqs, a.heads, a.dim, rest < blocks ? rest : blocks, join, true, false, 1.0);
        const Guess whole = brief ? guess(rows, a.n_seqs, a.heads, a.dim, blocks, join, false, false, share) : own;    // as the two parts are
        const Guess common = guess(all, 1, a.heads, a.dim, args->shared, join, true, false, 1.0, &left, (double)a.n_seqs * a.heads);
        if (common.us < whole.us) {
            ba_kv_scored_args s = *args;
            s.a.n_splits = left.parts;
            s.tile = left.v.rows;
            s.shared_parts = common.parts;
            s.shared_tile = common.v.rows;
            if (can_be_made(s)) {
                *args = s;
                return;
            }
        }
        args->shared = args->shared_parts = 0;
    }
    if (!can_be_made(*args)) {                               // one part, in the largest tiles: what the chip is full of anyway
        a.n_splits = 1;
        args->tile = 0;
    }
}

extern "C" int ba_kv_attend_scored(const ba_kv_scored_args* args, void* stream) {
    clear_error();
    BA_REQUIRE(args != nullptr, "null args");
    const ba_kv_scored_args& s = *args;
    bool nothing;
    const int rc = attend_check(s.a, nothing);
    if (rc != BA_OK) return rc;
    BA_REQUIRE(s.cap == 0.0f || (s.cap >= 1.0e-3f && s.cap <= 1.0e3f), "attention: cap must be in [1e-3, 1e3]");
    BA_REQUIRE(s.shared >= 0 && s.shared <= s.a.n_pages, "attention: shared blocks past the lists");
    BA_REQUIRE(s.shared ? s.shared_parts >= 1 && s.shared_parts <= 65536 : s.shared_parts == 0, "attention: bad shared_parts");
    BA_REQUIRE(s.a.n_splits + s.shared_parts <= 65536, "attention: too many parts");
    for (const int tile : {s.tile, s.shared_tile})
        BA_REQUIRE(tile == 0 || tile == 16 || tile == 32 || tile == 128 || (tile == 256 && s.a.dim <= 128), "attention: tiles have 16, 32, 128 or (up to heads of 128) 256 rows");
    if (nothing) return BA_OK;
    return attend_scored(s, (hipStream_t)stream);
}
