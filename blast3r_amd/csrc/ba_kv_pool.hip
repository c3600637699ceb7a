// Pages of the 8-bit key/value cache: which blocks the sequences' lists hold, kept on the device.
//
// A pool knows of each block how many lists hold it (counts) and, in a bit each, whether any does (used).  Blocks are taken
// lowest first and sequences served in their order, so every call has one result whatever order its threads run in:
// counts change by integer additions, which commute, and who gets which block comes of prefix sums.
//
//   count    counts from the lists
//   fork     children get their parents' lists: counts rise, nothing is copied
//   grow     blocks for new tokens.  An open last block that other lists hold too is exchanged for a block of one's own, with
//            the pair (old, new) to be copied; sequence after sequence, so that the last of its holders keeps it.
//   trim     blocks outside a range of tokens are given back
//   compact  the highest used blocks go to the lowest free ones
//   copy     blocks' codes and factors, pair by pair
//
// All but copy are a few thousand integers: their time is launches and dependent loads (lengths, lists, counts).  grow and
// the plan of compact run in one workgroup, where a barrier takes the place of a launch; bits in the place of counts make
// what it has to look through short (a million blocks are 128 KB).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ba_error.h"
#include "ba_hip.h"

namespace ba {

#define PL_T 256
#define PL_ONE 1024          // threads of the kernels that run in one workgroup

// what other threads of this launch change by atomics is read past the first cache
__device__ __forceinline__ int32_t fresh(const int32_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

__device__ __forceinline__ bool held(const ba_kv_pool& p, int32_t block) { return block >= 0 && block < p.n_blocks; }

__device__ __forceinline__ void hold(const ba_kv_pool& p, int32_t block) {
    if (atomicAdd(p.counts + block, 1) == 0) atomicOr(p.used + (block >> 5), 1u << (block & 31));
}

__device__ __forceinline__ void give_back(const ba_kv_pool& p, int32_t block) {
    const int32_t before = atomicSub(p.counts + block, 1);
    if (before == 1) atomicAnd(p.used + (block >> 5), ~(1u << (block & 31)));
    else if (before <= 0) atomicAdd(p.counts + block, 1);    // of no list that the pool knows
}

// ------------------------------------------------------------------------------------------------ counts from the lists

__global__ void __launch_bounds__(PL_T) k_pool_clear(ba_kv_pool p) {
    const int64_t i = (int64_t)blockIdx.x * PL_T + threadIdx.x;
    if (i >= p.n_blocks) return;
    p.counts[i] = 0;
    p.marks[i] = -1;
}

__global__ void __launch_bounds__(PL_T) k_pool_count(ba_kv_pool p, ba_kv_table t) {
    const int64_t n = (int64_t)t.n_seqs * t.n_pages;
    for (int64_t i = (int64_t)blockIdx.x * PL_T + threadIdx.x; i < n; i += (int64_t)gridDim.x * PL_T) {
        const int64_t s = i / t.n_pages;
        const int32_t b = t.pages[s * t.stride + (i - s * t.n_pages)];
        if (held(p, b)) atomicAdd(p.counts + b, 1);
    }
}

// a word of bits to a thread; those past the last block count as used
__global__ void __launch_bounds__(PL_T) k_pool_bits(ba_kv_pool p) {
    const int64_t w = (int64_t)blockIdx.x * PL_T + threadIdx.x;
    if (w >= (p.n_blocks + 31) / 32) return;
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const int64_t b = w * 32 + i;
        if (b >= p.n_blocks || p.counts[b] > 0) bits |= 1u << i;
    }
    p.used[w] = bits;
}

// ------------------------------------------------------------------------------------------------ lists forked, blocks given back

__global__ void __launch_bounds__(PL_T) k_pool_fork(ba_kv_pool p, ba_kv_fork_args a, int same) {
    const int i = blockIdx.x;
    const int32_t from = a.parents[i], to = a.children[i];
    if (from < 0 || from >= a.from.n_seqs || to < 0 || to >= a.to.n_seqs) return;
    // a child that a later pair has too, or that is a parent itself, is left as it is
    int out = 0;
    for (int j = threadIdx.x; j < a.n; j += PL_T) {
        if (j > i && a.children[j] == to) out = 1;
        if (same && a.parents[j] == to) out = 1;
    }
    if (__syncthreads_or(out)) return;
    const int32_t len = a.from_lengths[from];
    const int32_t* src = a.from.pages + from * a.from.stride;
    int32_t* dst = a.to.pages + to * a.to.stride;
    for (int b = threadIdx.x; b < a.to.n_pages; b += PL_T) {
        const int32_t old = dst[b];
        int32_t now = b < a.from.n_pages && (int64_t)b * 64 < len ? src[b] : -1;
        if (held(p, now)) hold(p, now);
        else now = -1;
        if (held(p, old)) give_back(p, old);
        if (now != old) dst[b] = now;
    }
    if (threadIdx.x == 0) a.to_lengths[to] = len;
}

// Rows of a table (those of the list `rows`, or all): what lies outside the tokens [first, last) is given back.
__global__ void __launch_bounds__(PL_T) k_pool_trim(ba_kv_pool p, ba_kv_trim_args a) {
    const int32_t s = a.rows ? a.rows[blockIdx.x] : (int32_t)blockIdx.x;
    if (s < 0 || s >= a.table.n_seqs) return;
    const int32_t first = a.first ? a.first[s] : 0, last = a.last ? a.last[s] : 0x7fffffff;
    const int64_t lo = first < 0 ? 0 : first / 64, hi = a.all ? 0 : last < 0 ? 0 : ((int64_t)last + 63) / 64;
    int32_t* row = a.table.pages + s * a.table.stride;
    for (int b = threadIdx.x; b < a.table.n_pages; b += PL_T) {
        if (b >= lo && b < hi) continue;
        if (row[b] < 0) continue;
        const int32_t old = atomicExch(row + b, -1);         // a row that is named twice gives back once
        if (held(p, old)) give_back(p, old);
    }
    if (a.lengths && threadIdx.x == 0) a.lengths[s] = 0;
}

// ------------------------------------------------------------------------------------------------ one workgroup

// sum of the values of the threads before this one, and of all; red: an int of LDS for each wave
__device__ __forceinline__ int scan_before(int v, int* red, int& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
        const int y = __shfl_up(x, k);
        if (lane >= k) x += y;
    }
    __syncthreads();                                         // red may still be read from the last call
    if (lane == 63) red[wave] = x;
    __syncthreads();
    int before = x - v;
    all = 0;
#pragma unroll
    for (int w = 0; w < PL_ONE / 64; ++w) {
        const int r = red[w];
        if (w < wave) before += r;
        all += r;
    }
    return before;
}

// The first `most` blocks that are free (want = false: ascending) or used (descending), in `list`; how many there are of them.
template <bool USED>
__device__ int pool_list(const ba_kv_pool& p, int32_t* list, int most, int* red) {
    const int words = (int)((p.n_blocks + 31) / 32);
    int found = 0;
    for (int base = 0; base < words && found < most; base += PL_ONE) {
        const int i = base + (int)threadIdx.x, w = USED ? words - 1 - i : i;
        uint32_t bits = 0;
        if (i < words) {
            bits = p.used[w];
            if (!USED) bits = ~bits;
            else if (w == words - 1 && p.n_blocks % 32) bits &= (1u << (p.n_blocks % 32)) - 1u;
        }
        int all, at = found + scan_before(__popc(bits), red, all);
        while (bits && at < most) {
            const int b = USED ? 31 - __clz(bits) : __ffs(bits) - 1;
            bits &= ~(1u << b);
            list[at++] = w * 32 + b;
        }
        found += all;
    }
    return found < most ? found : most;
}

// Sequences of a round have 1 << shift threads each, which take their new blocks side by side.
__global__ void __launch_bounds__(PL_ONE) k_pool_grow(ba_kv_pool p, ba_kv_grow_args a, int shift, int most) {
    __shared__ int red[PL_ONE / 64];
    const int tid = threadIdx.x, lanes = 1 << shift, l = tid & (lanes - 1), lead = (tid & 63) & ~(lanes - 1), per = PL_ONE >> shift;
    int32_t* list = p.marks + p.n_blocks;
    struct Seq {
        int len, filled, end;                                // blocks [filled, end) are those of new tokens alone
        int32_t open;                                        // the block that holds tokens and gets new ones, or -1
        int32_t* row;
    };
    auto seq = [&](int s) {
        Seq r = {0, 0, 0, -1, nullptr};
        if (s >= a.table.n_seqs) return r;
        const int64_t len = a.lengths[s] < 0 ? 0 : a.lengths[s];
        int64_t n = a.more ? a.more[s] : a.each;
        n = n < 0 ? 0 : n < a.max_new ? n : a.max_new;
        const int64_t end = (len + n + 63) / 64, filled = (len + 63) / 64;
        r.row = a.table.pages + s * a.table.stride;
        r.len = (int)len;
        r.end = (int)(end < a.table.n_pages ? end : a.table.n_pages);
        r.filled = (int)(filled < r.end ? filled : r.end);
        if (n > 0 && len % 64 && len / 64 < a.table.n_pages) r.open = r.row[len / 64];
        if (!held(p, r.open)) r.open = -1;
        return r;
    };
    // open blocks that other lists hold too: marked with the last sequence that is to write there, and given back by all
    int any = 0;
    for (int s = tid; s < a.table.n_seqs; s += PL_ONE) {
        const Seq r = seq(s);
        if (r.open < 0 || fresh(p.counts + r.open) < 2) continue;
        atomicMax(p.marks + r.open, s);
        any = 1;
    }
    any = __syncthreads_or(any);
    if (any) {
        for (int s = tid; s < a.table.n_seqs; s += PL_ONE) {
            const Seq r = seq(s);
            if (r.open >= 0 && fresh(p.marks + r.open) >= 0) atomicSub(p.counts + r.open, 1);
        }
    }
    const int free = pool_list<false>(p, list, most, red);
    __syncthreads();
    int base = 0, moves = 0;
    for (int s0 = 0; s0 < a.table.n_seqs; s0 += per) {
        const int s = s0 + (tid >> shift);
        const Seq r = seq(s);
        // the last holder of a block that no other list holds any more keeps it
        bool own = false, final = false, keeps = false;
        if (any && r.open >= 0) {
            const int last = fresh(p.marks + r.open);
            final = last == s;
            keeps = final && fresh(p.counts + r.open) == 0;
            own = last >= 0 && !keeps;
        }
        const unsigned long long mine = (lanes == 64 ? ~0ull : (1ull << lanes) - 1ull) << lead;
        int wants = own ? 1 : 0;
        for (int b = r.filled; __any(b < r.end); b += lanes) {
            const bool want = b + l < r.end && r.row[b + l] < 0;
            wants += __popcll(__ballot(want) & mine);
        }
        int all;
        int at = base + scan_before(l == 0 ? wants : 0, red, all);
        at = __shfl(at, lead);
        base += all;
        int32_t got = -1;
        if (own) {
            got = at < free ? list[at] : -1;
            ++at;
        }
        for (int b = r.filled; __any(b < r.end); b += lanes) {
            const bool want = b + l < r.end && r.row[b + l] < 0;
            const unsigned long long who = __ballot(want) & mine;
            if (want) {
                const int k = at + __popcll(who & ((1ull << (tid & 63)) - 1ull));
                if (k < free) {
                    const int32_t block = list[k];
                    r.row[b + l] = block;
                    p.counts[block] = 1;
                    atomicOr(p.used + (block >> 5), 1u << (block & 31));
                } else if (r.row[b + l] != -1) {
                    r.row[b + l] = -1;
                }
            }
            at += __popcll(who);
        }
        if (!any) continue;
        int made;
        const int m = moves + scan_before(l == 0 && got >= 0 ? 1 : 0, red, made);
        moves += made;
        // (all threads of the round have read marks and counts before the scans)
        if (l == 0 && final) p.marks[r.open] = -1;
        if (l == 0 && keeps) p.counts[r.open] = 1;
        if (l == 0 && own) {
            r.row[r.len / 64] = got;
            if (got >= 0) {
                a.src[m] = r.open;
                a.dst[m] = got;
                p.counts[got] = 1;
                atomicOr(p.used + (got >> 5), 1u << (got & 31));
            }
        }
    }
    for (int m = moves + tid; m < a.table.n_seqs; m += PL_ONE) {
        a.src[m] = -1;
        a.dst[m] = -1;
    }
    if (tid == 0) {
        *a.n = moves;
        *a.missing = base > free ? base - free : 0;
    }
}

// The k-th highest used block is to go to the k-th lowest free one while that is lower: as many pairs as there are used blocks
// past the number of used ones.
__global__ void __launch_bounds__(PL_ONE) k_pool_plan(ba_kv_pool p, int32_t* src, int32_t* dst, int32_t* n, int most) {
    __shared__ int red[PL_ONE / 64];
    const int tid = threadIdx.x, words = (int)((p.n_blocks + 31) / 32), spare = (int)((int64_t)words * 32 - p.n_blocks);
    int v = 0, total, above;
    for (int w = tid; w < words; w += PL_ONE) v += __popc(p.used[w]);
    if (tid == 0) v -= spare;
    scan_before(v, red, total);                              // used blocks
    v = 0;
    for (int w = total / 32 + tid; w < words; w += PL_ONE) {
        uint32_t bits = p.used[w];
        if (w == total / 32) bits &= ~0u << (total % 32);
        v += __popc(bits);
    }
    if (tid == 0) v -= spare;                                // its word is among them if there are any
    scan_before(v, red, above);
    const int pairs = above < most ? above : most;
    pool_list<false>(p, dst, pairs, red);
    pool_list<true>(p, src, pairs, red);
    __syncthreads();
    for (int k = tid; k < most; k += PL_ONE) {
        if (k >= pairs) {
            src[k] = -1;
            dst[k] = -1;
            continue;
        }
        const int32_t a = src[k], b = dst[k];
        p.counts[b] = p.counts[a];
        p.counts[a] = 0;
        p.marks[a] = b;
        atomicOr(p.used + (b >> 5), 1u << (b & 31));
        atomicAnd(p.used + (a >> 5), ~(1u << (a & 31)));
    }
    if (tid == 0) *n = pairs;
}

// entries of lists whose block moves
__global__ void __launch_bounds__(PL_T) k_pool_move(ba_kv_pool p, ba_kv_table t) {
    const int64_t n = (int64_t)t.n_seqs * t.n_pages;
    for (int64_t i = (int64_t)blockIdx.x * PL_T + threadIdx.x; i < n; i += (int64_t)gridDim.x * PL_T) {
        const int64_t s = i / t.n_pages;
        int32_t* e = t.pages + s * t.stride + (i - s * t.n_pages);
        const int32_t b = *e;
        if (!held(p, b)) continue;
        const int32_t to = p.marks[b];
        if (to >= 0) *e = to;
    }
}

__global__ void __launch_bounds__(PL_T) k_pool_unmark(ba_kv_pool p, const int32_t* src, int most) {
    const int k = blockIdx.x * PL_T + threadIdx.x;
    if (k < most && src[k] >= 0) p.marks[src[k]] = -1;
}

// ------------------------------------------------------------------------------------------------ blocks copied

#define CP_UNITS 1024        // pieces of 16 bytes that a workgroup copies at a time: 4 to a thread

// Workgroups take the pieces of all pairs in turn.
__global__ void __launch_bounds__(PL_T) k_kv_copy(ba_kv_copy_args a, int units, int chunks) {
    int n = a.n;
    if (a.count) {
        const int c = *a.count;
        n = c < n ? c : n;
    }
    const int per = 2 * chunks;
    for (int64_t item = blockIdx.x; item < (int64_t)n * per; item += gridDim.x) {
        const int pair = (int)(item / per), part = (int)(item - (int64_t)pair * per), chunk = part >> 1;
        const int32_t from = a.src[pair], to = a.dst[pair];
        if (from < 0 || from >= a.n_blocks || to < 0 || to >= a.n_blocks || from == to) continue;
        uint8_t* base = (uint8_t*)(part & 1 ? a.v : a.k);
        const uint4* x = (const uint4*)(base + (int64_t)from * units * 16);
        uint4* y = (uint4*)(base + (int64_t)to * units * 16);
        uint4 w[CP_UNITS / PL_T];
#pragma unroll
        for (int i = 0; i < CP_UNITS / PL_T; ++i) {
            const int u = chunk * CP_UNITS + i * PL_T + (int)threadIdx.x;
            if (u < units) w[i] = x[u];
        }
        if (part == 0)
            for (int h = threadIdx.x; h < 2 * a.heads; h += PL_T) a.scales[(int64_t)to * 2 * a.heads + h] = a.scales[(int64_t)from * 2 * a.heads + h];
#pragma unroll
        for (int i = 0; i < CP_UNITS / PL_T; ++i) {
            const int u = chunk * CP_UNITS + i * PL_T + (int)threadIdx.x;
            if (u < units) y[u] = w[i];
        }
    }
}

static int pool_check(const ba_kv_pool& p) {
    BA_REQUIRE(p.n_blocks >= 0 && p.n_blocks < (int64_t)1 << 30, "pool: bad sizes");
    BA_REQUIRE(p.n_blocks == 0 || (p.counts && p.used && p.marks), "null pointer");
    return BA_OK;
}

static int table_check(const ba_kv_table& t) {
    BA_REQUIRE(t.n_seqs >= 0 && t.n_pages >= 0 && t.n_pages < 1 << 24, "pool: bad sizes");
    BA_REQUIRE(t.n_seqs < 1 << 23, "pool: too many lists");
    BA_REQUIRE(t.n_seqs == 0 || t.n_pages == 0 || t.pages, "null pointer");
    return BA_OK;
}

static unsigned entry_grid(const ba_kv_table& t) {
    const int64_t nb = ((int64_t)t.n_seqs * t.n_pages + PL_T - 1) / PL_T;
    return (unsigned)(nb < 4096 ? nb : 4096);
}

}  // namespace ba

using namespace ba;

#define POOL_TRY(call) do { const int rc_ = (call); if (rc_ != BA_OK) return rc_; } while (0)

extern "C" int ba_kv_pool_count(const ba_kv_pool* pool, const ba_kv_table* tables, int32_t n_tables, void* stream) {
    clear_error();
    BA_REQUIRE(pool != nullptr && n_tables >= 0 && (n_tables == 0 || tables), "null args");
    POOL_TRY(pool_check(*pool));
    for (int i = 0; i < n_tables; ++i) POOL_TRY(table_check(tables[i]));
    if (pool->n_blocks == 0) return BA_OK;
    hipStream_t st = (hipStream_t)stream;
    const ba_kv_pool p = *pool;
    const unsigned nb = (unsigned)((p.n_blocks + PL_T - 1) / PL_T);
    hipLaunchKernelGGL(k_pool_clear, dim3(nb), dim3(PL_T), 0, st, p);
    for (int i = 0; i < n_tables; ++i)
        if (tables[i].n_seqs && tables[i].n_pages) hipLaunchKernelGGL(k_pool_count, dim3(entry_grid(tables[i])), dim3(PL_T), 0, st, p, tables[i]);
    hipLaunchKernelGGL(k_pool_bits, dim3((nb + 31) / 32), dim3(PL_T), 0, st, p);
    BA_LAUNCHED();
    return BA_OK;
}

extern "C" int ba_kv_pool_fork(const ba_kv_pool* pool, const ba_kv_fork_args* args, void* stream) {
    clear_error();
    BA_REQUIRE(pool && args, "null args");
    const ba_kv_fork_args& a = *args;
    POOL_TRY(pool_check(*pool));
    POOL_TRY(table_check(a.from));
    POOL_TRY(table_check(a.to));
    BA_REQUIRE(a.n >= 0 && a.n < 1 << 23, "pool: bad sizes");
    BA_REQUIRE(a.to.n_pages >= a.from.n_pages, "pool: children's lists are narrower than their parents'");
    if (a.n == 0 || a.from.n_seqs == 0 || a.to.n_seqs == 0) return BA_OK;
    BA_REQUIRE(a.parents && a.children && a.from_lengths && a.to_lengths, "null pointer");
    hipLaunchKernelGGL(k_pool_fork, dim3((unsigned)a.n), dim3(PL_T), 0, (hipStream_t)stream, *pool, a, (int)(a.from.pages == a.to.pages));
    BA_LAUNCHED();
    return BA_OK;
}

extern "C" int ba_kv_pool_trim(const ba_kv_pool* pool, const ba_kv_trim_args* args, void* stream) {
    clear_error();
    BA_REQUIRE(pool && args, "null args");
    const ba_kv_trim_args& a = *args;
    POOL_TRY(pool_check(*pool));
    POOL_TRY(table_check(a.table));
    BA_REQUIRE(a.n_rows >= 0 && a.n_rows < 1 << 23, "pool: bad sizes");
    const int n = a.rows ? a.n_rows : a.table.n_seqs;
    if (n == 0 || a.table.n_seqs == 0) return BA_OK;
    hipLaunchKernelGGL(k_pool_trim, dim3((unsigned)n), dim3(PL_T), 0, (hipStream_t)stream, *pool, a);
    BA_LAUNCHED();
    return BA_OK;
}

extern "C" int ba_kv_pool_grow(const ba_kv_pool* pool, const ba_kv_grow_args* args, void* stream) {
    clear_error();
    BA_REQUIRE(pool && args, "null args");
    const ba_kv_grow_args& a = *args;
    POOL_TRY(pool_check(*pool));
    POOL_TRY(table_check(a.table));
    BA_REQUIRE(a.max_new >= 0, "pool: bad sizes");
    BA_REQUIRE(a.n && a.missing && (a.table.n_seqs == 0 || (a.lengths && a.src && a.dst)), "null pointer");
    // blocks that a sequence may need: threads for as many, and a list of what all of them may take
    int64_t slots = ((int64_t)a.max_new + 63) / 64;
    slots = slots < a.table.n_pages ? slots : a.table.n_pages;
    int shift = 0;
    while (shift < 6 && (1 << shift) < slots) ++shift;
    const int64_t most = (slots + 1) * a.table.n_seqs;
    hipLaunchKernelGGL(k_pool_grow, dim3(1), dim3(PL_ONE), 0, (hipStream_t)stream, *pool, a, shift, (int)(most < pool->n_blocks ? most : pool->n_blocks));
    BA_LAUNCHED();
    return BA_OK;
}

extern "C" int ba_kv_pool_compact(const ba_kv_pool* pool, const ba_kv_table* tables, int32_t n_tables, int32_t* src, int32_t* dst,
                                  int32_t* n, int32_t most, void* stream) {
    clear_error();
    BA_REQUIRE(pool != nullptr && n_tables >= 0 && (n_tables == 0 || tables), "null args");
    POOL_TRY(pool_check(*pool));
    for (int i = 0; i < n_tables; ++i) POOL_TRY(table_check(tables[i]));
    BA_REQUIRE(most >= 0 && most <= pool->n_blocks, "pool: bad sizes");
    BA_REQUIRE(n && (most == 0 || (src && dst)), "null pointer");
    hipStream_t st = (hipStream_t)stream;
    const ba_kv_pool p = *pool;
    hipLaunchKernelGGL(k_pool_plan, dim3(1), dim3(PL_ONE), 0, st, p, src, dst, n, most);
    if (most) {
        for (int i = 0; i < n_tables; ++i)
            if (tables[i].n_seqs && tables[i].n_pages) hipLaunchKernelGGL(k_pool_move, dim3(entry_grid(tables[i])), dim3(PL_T), 0, st, p, tables[i]);
        hipLaunchKernelGGL(k_pool_unmark, dim3((unsigned)((most + PL_T - 1) / PL_T)), dim3(PL_T), 0, st, p, src, most);
    }
    BA_LAUNCHED();
    return BA_OK;
}

extern "C" int ba_kv_copy(const ba_kv_copy_args* args, void* stream) {
    clear_error();
    BA_REQUIRE(args != nullptr, "null args");
    const ba_kv_copy_args& a = *args;
    BA_REQUIRE(a.n_blocks >= 0 && a.heads >= 1 && a.heads <= 65536 && a.n >= 0, "cache: bad sizes");
    BA_REQUIRE(a.dim == 32 || a.dim == 64 || a.dim == 96 || a.dim == 128 || a.dim == 256,
               "cache: head size must be 32, 64, 96, 128 or 256");
    if (a.n == 0 || a.n_blocks == 0) return BA_OK;
    BA_REQUIRE(a.k && a.v && a.scales && a.src && a.dst, "null pointer");
    BA_REQUIRE((uintptr_t)a.k % 16 == 0 && (uintptr_t)a.v % 16 == 0, "cache: k and v must be aligned to 16 bytes");
    const int units = a.heads * a.dim * 4, chunks = (units + CP_UNITS - 1) / CP_UNITS;
    const int64_t items = (int64_t)a.n * 2 * chunks;
    hipLaunchKernelGGL(k_kv_copy, dim3((unsigned)(items < 4096 ? items : 4096)), dim3(PL_T), 0, (hipStream_t)stream, a, units, chunks);
    BA_LAUNCHED();
    return BA_OK;
}
