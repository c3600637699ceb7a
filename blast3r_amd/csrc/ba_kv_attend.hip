// Attention over the 8-bit key/value cache: the plain form, and what its kernels share with the others (ba_kv_attend.h).
#include <math.h>

#include "ba_kv_attend.h"

using namespace ba;

extern "C" int32_t ba_kv_attend_splits(int32_t n_seqs, int32_t heads, int32_t q_heads, int32_t dim, int64_t max_rows,
                                       int32_t n_pages) {
    if (n_seqs < 1 || heads < 1 || q_heads < heads || max_rows < 1 || n_pages < 1 || dim < 4) return 1;
    const int64_t rows = max_rows * (q_heads / heads);
    const AtShape v = at_shape(rows, dim);
    // two parts of so many workgroups, or the join of so many rows, are more than a launch can have
    const double most_rows = ((1 << 24) - 1) * (double)(AT_T / (dim / 4)), all_rows = (double)n_seqs * max_rows * q_heads;
    if ((double)n_seqs * heads * ceil((double)rows / v.rows) >= 1 << 22 || all_rows > most_rows || all_rows >= 2147483648.0) return 1;
    const int64_t base = (int64_t)n_seqs * heads * ((rows + v.rows - 1) / v.rows);
    const int64_t most = (n_pages + AT_MIN_BLOCKS - 1) / AT_MIN_BLOCKS;
    // Many rows: as many workgroups as the CUs hold at a time.  Few rows read memory: one and a half per CU do, and
    // at least two parts for sequences of different lengths.
    int64_t n = v.ncb ? 256 * v.fit / base : (384 + base - 1) / base;
    if (v.ncb == 0 && n < 2) n = 2;
    n = n < most ? n : most;
    return (int32_t)(n < 1 ? 1 : n);
}

extern "C" int64_t ba_kv_attend_workspace_bytes(int64_t n_rows, int32_t q_heads, int32_t dim, int32_t n_splits) {
    return n_splits > 1 && n_rows > 0 ? n_rows * q_heads * n_splits * ((int64_t)dim + 2) * 4 : 0;
}

// What every attention call is checked for, before anything is launched; `nothing`: it has no rows.
int ba::attend_check(const ba_kv_attend_args& a, bool& nothing) {
    nothing = false;
    BA_REQUIRE(a.n_blocks >= 0 && a.n_blocks <= KV_KEPT && a.heads >= 1 && a.heads <= 65536 && a.n_seqs >= 0 && a.n_pages >= 0, "attention: bad sizes");
    BA_REQUIRE(a.dim == 32 || a.dim == 64 || a.dim == 96 || a.dim == 128 || a.dim == 256,
               "attention: head size must be 32, 64, 96, 128 or 256");
    BA_REQUIRE(a.q_heads >= 1 && a.q_heads <= 65536 && a.q_heads % a.heads == 0, "attention: query heads must be a multiple of the cache's");
    BA_REQUIRE(a.bits == BA_FP8 || a.bits == BA_INT8, "attention: bits must be 0 (e4m3) or 1 (int8)");
    BA_REQUIRE(a.dtype == BA_F16 || a.dtype == BA_BF16, "attention: queries must be fp16 or bf16");
    BA_REQUIRE(a.n_rows >= 0 && a.rows_per_seq >= 0 && a.max_rows >= 0 && a.window >= 0 && a.n_rows < (int64_t)1 << 31 &&
                   a.max_rows < (int64_t)1 << 31 && a.rows_per_seq < (int64_t)1 << 31 && a.n_pages < 1 << 24, "attention: bad sizes");
    BA_REQUIRE(a.scale > 0.0f && a.scale < 1.0e30f, "attention: scale must be positive");
    BA_REQUIRE(a.n_splits >= 1 && a.n_splits <= 65536, "attention: n_splits must be in [1, 65536]");
    nothing = a.n_rows == 0 || a.n_seqs == 0 || a.max_rows == 0;
    if (nothing) return BA_OK;
    BA_REQUIRE(a.offsets != nullptr || a.rows_per_seq >= 1, "attention: rows without sequences");
    BA_REQUIRE(a.q && a.o && a.lengths, "null pointer");
    BA_REQUIRE((a.n_pages == 0 || a.pages) && (a.n_blocks == 0 || (a.k && a.v && a.scales)), "null pointer");
    BA_REQUIRE((uintptr_t)a.k % 16 == 0 && (uintptr_t)a.v % 16 == 0 && (uintptr_t)a.scales % 8 == 0,
               "attention: k and v must be aligned to 16 bytes, scales to 8");
    return BA_OK;
}

// The workgroups of a launch over `rows` (query rows times the heads that share a cache head) of each of n_seqs sequences.
int ba::attend_grid(const ba_kv_attend_args& a, int64_t rows, int64_t n_seqs, int parts, const AtShape& v, AtGrid& g) {
    const int tile = v.rows;
    BA_REQUIRE(rows < ((int64_t)1 << 31) - 256, "attention: too many rows for a call");
    int64_t tiles = (rows + tile - 1) / tile, per_tile = n_seqs * a.heads * parts;
    // a launch has less than 2^32 threads, 512 to a workgroup
    const int64_t most = ((int64_t)1 << 23) - 1;
    const bool packed = a.offsets && n_seqs > 1 && tiles > most / per_tile;
    if (packed) {
        tiles = a.n_rows * (a.q_heads / a.heads) / tile + n_seqs;
        per_tile = (int64_t)a.heads * parts;
    }
    BA_REQUIRE(tiles <= most / per_tile, "attention: too many tiles for a call");
    g = {(unsigned)(tiles * per_tile), (int)tiles, (int)packed};
    return BA_OK;
}

// The join of the parts: those of a row are shared among threads while the chip has room for more of them.
int ba::attend_join(const ba_kv_attend_args& a, AtJoin& j) {
    const int64_t jobs = a.n_rows * a.q_heads;
    j = {1, 0};
    if (a.n_splits == 1) return BA_OK;
    while (j.lanes < a.n_splits && 2 * j.lanes * (a.dim / 4) <= AT_T && jobs * (a.dim / 4) * j.lanes < 256 * 1024) j.lanes *= 2;
    const int per_wg = AT_T / (a.dim / 4) / j.lanes;
    // (which keeps the bytes of the workspace below 2^58 too)
    BA_REQUIRE(jobs < (int64_t)1 << 31 && (jobs + per_wg - 1) / per_wg < (int64_t)1 << 24, "attention: too many rows for a call");
    BA_REQUIRE(a.workspace && (uintptr_t)a.workspace % 16 == 0, "null pointer");
    BA_REQUIRE(a.workspace_bytes >= ba_kv_attend_workspace_bytes(a.n_rows, a.q_heads, a.dim, a.n_splits), "attention: workspace too small");
    j.nb = (unsigned)((jobs + per_wg - 1) / per_wg);
    return BA_OK;
}

// loads of 8 queries, stores of 4 outputs
int ba::attend_wide(const ba_kv_attend_args& a) {
    return (uintptr_t)a.q % 16 == 0 && (uintptr_t)a.o % 8 == 0 && a.q_st % 8 == 0 && a.q_sh % 8 == 0 && a.o_st % 4 == 0 && a.o_sh % 4 == 0;
}

extern "C" int ba_kv_attend(const ba_kv_attend_args* args, void* stream) {
    clear_error();
    BA_REQUIRE(args != nullptr, "null args");
    ba_kv_attend_args a = *args;
    bool nothing;
    int rc = attend_check(a, nothing);
    if (rc != BA_OK || nothing) return rc;
    a.window = at_window(a.window);
    const int64_t rows = a.max_rows * (a.q_heads / a.heads);
    const AtShape v = at_shape(rows, a.dim);
    AtGrid g;
    AtJoin j;
    rc = attend_grid(a, rows, a.n_seqs, a.n_splits, v, g);
    if (rc == BA_OK) rc = attend_join(a, j);
    if (rc != BA_OK) return rc;
    const int wide = attend_wide(a);
    hipStream_t st = (hipStream_t)stream;
    const AtArgs<AT_PLAIN> x = {a};
    rc = v.ncb ? launch_tiles<AT_PLAIN>(x, v, g, wide, st) : launch_few<AT_PLAIN>(x, v, g, wide, st);
    if (rc != BA_OK || a.n_splits == 1) return rc;
    hipLaunchKernelGGL(k_kv_join<AT_PLAIN>, dim3(j.nb), dim3(AT_T), 0, st, x, v.rows, j.lanes, wide);
    BA_LAUNCHED();
    return BA_OK;
}
