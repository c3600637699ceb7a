// Attention over the 8-bit cache with formed scores, masks by row and sequences that begin alike.
//
//   z_j = scale q.k_j;  with a cap: cap tanh(z_j / cap);  with slopes: less slope |p - j|
//   o = sum_j e^z_j v_j / sum_j e^z_j  over the tokens j that a row sees:
//   j < prefix of its sequence, or since <= j < until of the row, causal and in the window
//
// The kernels are those of ba_kv_attend.h.  What a row sees is two intervals there (AtRow), and a workgroup walks over the
// blocks that any of its rows sees (AtWalk): a window behind a prefix, or a document in a long prompt, costs its own blocks.
//
// shared: the first so many blocks of all lists are the same.  One launch takes the rows of all sequences over these blocks as
// if they were one sequence's (AtMore.stacked), another each sequence's own blocks, and both leave partial sums for one join:
// the shared tokens are read, and converted, once for up to 256 rows instead of once for each sequence.
#include "ba_kv_attend.h"

namespace ba {

extern template int launch_attend<AT_SLOPES>(const AtArgs<AT_SLOPES>&, AtShape, unsigned, int, int, int, hipStream_t);
extern template int launch_attend<AT_CAPPED>(const AtArgs<AT_CAPPED>&, AtShape, unsigned, int, int, int, hipStream_t);

template <int MODE>
static int attend_scored(const ba_kv_scored_args& s, hipStream_t st) {
    AtArgs<MODE> x;
    x.a = s.a;
    x.a.n_splits = s.a.n_splits + s.shared_parts;
    const int group = s.a.q_heads / s.a.heads;
    const int64_t rows = s.a.max_rows * group, all = s.a.n_rows * group;
    const AtShape v = at_shape(rows, s.a.dim), w = at_shape(all, s.a.dim);
    AtGrid g, h;
    AtJoin j;
    int rc = attend_grid(x.a, rows, s.a.n_seqs, s.a.n_splits, v, g);
    if (rc == BA_OK && s.shared) rc = attend_grid(x.a, all, 1, s.shared_parts, w, h);
    if (rc == BA_OK) rc = attend_join(x.a, j);
    if (rc != BA_OK) return rc;
    const int wide = attend_wide(s.a);
    x.m = {s.slopes, s.prefix, s.since, s.until, s.cap, 0, s.shared, 0, s.shared_parts, 1};
    if (s.shared) rc = launch_attend<MODE>(x, w, h.nb, h.tiles, h.packed, wide, st);
    if (rc != BA_OK) return rc;
    x.m.blk_lo = s.shared;
    x.m.blk_hi = s.a.n_pages;
    x.m.part0 = s.shared_parts;
    x.m.parts = s.a.n_splits;
    x.m.stacked = 0;
    rc = launch_attend<MODE>(x, v, g.nb, g.tiles, g.packed, wide, st);
    if (rc != BA_OK || x.a.n_splits == 1) return rc;
    hipLaunchKernelGGL(k_kv_join<MODE>, dim3(j.nb), dim3(AT_T), 0, st, x, v.rows, j.lanes, wide);
    BA_LAUNCHED();
    return BA_OK;
}

// Parts for a launch of `base` workgroups that may have `blocks` blocks each: as for the plain form.
static int parts_of(int64_t base, int64_t blocks, const AtShape& v, int least) {
    const int64_t most = (blocks + AT_MIN_BLOCKS - 1) / AT_MIN_BLOCKS;
    int64_t n = v.ncb ? 256 * v.fit / base : (384 + base - 1) / base;
    if (v.ncb == 0 && n < least) n = least;
    n = n < most ? n : most;
    return (int)(n < 1 ? 1 : n);
}

}  // namespace ba

using namespace ba;

extern "C" void ba_kv_scored_parts(const ba_kv_scored_args* args, int32_t* own, int32_t* shared) {
    const ba_kv_attend_args& a = args->a;
    *own = 1;
    *shared = args->shared > 0 ? 1 : 0;
    if (a.n_seqs < 1 || a.heads < 1 || a.q_heads < a.heads || a.max_rows < 1 || a.n_rows < 1 || args->shared < 0) return;
    const int group = a.q_heads / a.heads;
    const int64_t rows = a.max_rows * group, all = a.n_rows * group;
    const AtShape v = at_shape(rows, a.dim), w = at_shape(all, a.dim);
    int64_t blocks = a.n_pages - args->shared;
    if (a.window > 0 && !args->prefix) {                     // what a tile's rows can see
        const int64_t tile = v.rows / group < a.max_rows ? v.rows / group + 1 : a.max_rows, seen = (a.window + tile + 62) / 64 + 1;
        blocks = seen < blocks ? seen : blocks;
    }
    *own = parts_of((int64_t)a.n_seqs * a.heads * ((rows + v.rows - 1) / v.rows), blocks, v, 2);
    if (args->shared > 0) *shared = parts_of((int64_t)a.heads * ((all + w.rows - 1) / w.rows), args->shared, w, 1);
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
    if (nothing) return BA_OK;
    hipStream_t st = (hipStream_t)stream;
    if (s.cap != 0.0f) return attend_scored<AT_CAPPED>(s, st);
    return s.slopes ? attend_scored<AT_SLOPES>(s, st) : attend_scored<AT_MASKS>(s, st);
}
