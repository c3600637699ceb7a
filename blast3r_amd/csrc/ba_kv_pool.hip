// Pages of the 8-bit key/value cache: which blocks the sequences' lists hold, kept on the device.
//
// A pool knows of each block how many lists hold it (counts) and, in a bit each, whether any does (used).  Blocks are taken
// lowest first and sequences served in their order, so every call has one result whatever order its threads run in:
// counts change by integer additions, which commute, and who gets which block comes of prefix sums.
//
//   count    counts from the lists
//   fork     children get their parents' lists: counts rise, nothing is copied
//   grow     blocks for new tokens.  An open last block that other lists hold too is exchanged for a block of one's own, with
//            the pair (old, new) to be copied; sequence after sequence, so that the last of its holders keeps it.  Without
//            a block to exchange it for it stays, marked (KV_KEPT): its tokens are seen, and nothing is written there.
//   trim     blocks outside a range of tokens are given back
//   compact  the highest used blocks go to the lowest free ones
//   copy     blocks' codes and factors, pair by pair
//
// All but copy are a few thousand integers: their time is launches and dependent loads (lengths, lists, counts).  grow and
// the plan of compact run in one workgroup, where a barrier takes the place of a launch; bits in the place of counts make
// what it has to look through short (a million blocks are 128 KB).  For 64 to 128 sequences and 5000 blocks: count 4 us, fork
// 5.5, trim 3, grow 6 (9 where 120 open blocks are exchanged), the plan of 870 moves 6 and the lists 3.  copy is bound by
// memory: 870 blocks of 131 KB (228 MB read and written) 42 us, 5.4 TB/s, as a large copy.  Pairs of a fork are each compared with
// all others: 128 8 us with the launch, 8192 48, 65536 1.9 ms; lists of a grow go 1024 at a time: 16384 61 us, 131072 0.5 ms.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ba_error.h"
#include "ba_hip.h"
#include "ba_token.h"

namespace ba {

#define PL_T 256
#define PL_ONE 1024          // threads of the kernels that run in one workgroup
#define PL_FEW 16384         // blocks that one workgroup counts (64 KB), and half of the entries

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
        const int32_t b = kv_block(t.pages[s * t.stride + (i - s * t.n_pages)]);
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

// The same of one table in one launch, where that is little: counts are made in LDS.
__global__ void __launch_bounds__(PL_ONE) k_pool_count_one(ba_kv_pool p, ba_kv_table t) {
    extern __shared__ int32_t counts_sh[];
    const int blocks = (int)p.n_blocks, n = t.n_seqs * t.n_pages;
    for (int i = threadIdx.x; i < blocks; i += PL_ONE) counts_sh[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += PL_ONE) {
        const int s = (int)((unsigned)i / (unsigned)t.n_pages);
        const int32_t b = kv_block(t.pages[s * t.stride + (i - s * t.n_pages)]);
        if (held(p, b)) atomicAdd(counts_sh + b, 1);
    }
    __syncthreads();
    // a lane to a block, a ballot to two words
    for (int i = threadIdx.x; i < (blocks + 63) / 64 * 64; i += PL_ONE) {
        const int c = i < blocks ? counts_sh[i] : 1;
        if (i < blocks) {
            p.counts[i] = c;
            p.marks[i] = -1;
        }
        const unsigned long long bits = __ballot(c > 0);
        if ((i & 31) == 0 && i < (blocks + 31) / 32 * 32) p.used[i / 32] = (uint32_t)(i & 32 ? bits >> 32 : bits);
    }
}

// ------------------------------------------------------------------------------------------------ lists forked, blocks given back

__global__ void __launch_bounds__(PL_T) k_pool_fork(ba_kv_fork_args a, int same) {
    const ba_kv_pool& p = a.pool;
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
        const int32_t old = dst[b], given = kv_block(old);
        int32_t now = b < a.from.n_pages && (int64_t)b * 64 < len ? src[b] : -1;
        if (held(p, kv_block(now))) hold(p, kv_block(now));
        else now = -1;
        if (held(p, given)) give_back(p, given);
        if (now != old) dst[b] = now;
    }
    if (threadIdx.x == 0) a.to_lengths[to] = len;
}

// Rows of a table (those of the list `rows`, or all): what lies outside the tokens [first, last) is given back.
__global__ void __launch_bounds__(PL_T) k_pool_trim(ba_kv_trim_args a) {
    const ba_kv_pool& p = a.pool;
    const int32_t s = a.rows ? a.rows[blockIdx.x] : (int32_t)blockIdx.x;
    if (s < 0 || s >= a.table.n_seqs) return;
    const int32_t first = a.first ? a.first[s] : 0, last = a.last ? a.last[s] : 0x7fffffff;
    const int64_t lo = first < 0 ? 0 : first / 64, hi = a.all ? 0 : last < 0 ? 0 : ((int64_t)last + 63) / 64;
    int32_t* row = a.table.pages + s * a.table.stride;
    for (int b = threadIdx.x; b < a.table.n_pages; b += PL_T) {
        if (b >= lo && b < hi) continue;
        if (row[b] < 0) continue;
        const int32_t old = kv_block(atomicExch(row + b, -1));         // a row that is named twice gives back once
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

// Words of bits are looked through a thread each, then 32 threads take the bits of one (a thread that wrote all of its word's
// blocks was most of the time of a pool of 5000 of them: 19 us for the plan of its moves).  each(word, used bits, used blocks
// before it) in the order of the words, by 32 threads a word, until it has seen `enough` used (USED) or free blocks.
template <bool USED, typename F>
__device__ __forceinline__ void pool_words(const ba_kv_pool& p, int enough, int* red, uint2* words_sh, F each) {
    const int words = (int)((p.n_blocks + 31) / 32);
    int used = 0;
    for (int base = 0; base < words && (USED ? used : base * 32 - used) < enough; base += PL_ONE) {
        const int w = base + (int)threadIdx.x;
        uint32_t bits = 0;
        if (w < words) {
            bits = p.used[w];
            if (w == words - 1 && p.n_blocks % 32) bits &= (1u << (p.n_blocks % 32)) - 1u;
        }
        int all;
        const int at = used + scan_before(__popc(bits), red, all);
        words_sh[threadIdx.x] = make_uint2(bits, (uint32_t)at);      // (the scan has barriers: nobody reads the last round's)
        __syncthreads();
        const int here = min(words - base, PL_ONE);
        for (int k = threadIdx.x >> 5; k < here; k += PL_ONE / 32) {
            const uint2 x = words_sh[k];
            if ((USED ? (int)x.y : (base + k) * 32 - (int)x.y) >= enough) break;
            each(base + k, x.x, (int)x.y);
        }
        used += all;
    }
}

__global__ void __launch_bounds__(PL_ONE) k_pool_available(ba_kv_free_args a) {
    const ba_kv_pool& p = a.pool;
    __shared__ int red[PL_ONE / 64];
    const int words = (int)((p.n_blocks + 31) / 32);
    int v = 0, total;
    for (int w = threadIdx.x; w < words; w += PL_ONE) v += __popc(~p.used[w]);       // bits past the last block are set
    scan_before(v, red, total);
    if (threadIdx.x == 0) *a.free = total;
}

// The first `most` free blocks in `list`; how many there are of them.
__device__ int pool_free(const ba_kv_pool& p, int32_t* list, int most, int* red, uint2* words_sh, int* found_sh) {
    if (threadIdx.x == 0) *found_sh = 0;
    const int bit = threadIdx.x & 31;
    int found = 0;
    __syncthreads();
    pool_words<false>(p, most, red, words_sh, [&](int w, uint32_t used, int before) {
        const int64_t block = (int64_t)w * 32 + bit;
        const int at = w * 32 - before + __popc(~used & ((1u << bit) - 1u));
        if ((used >> bit & 1u) || block >= p.n_blocks || at >= most) return;
        list[at] = (int32_t)block;
        found = at + 1;
    });
    if (found) atomicMax(found_sh, found);
    __syncthreads();
    return *found_sh;
}

// Sequences of a round have 1 << shift threads each, which take their new blocks side by side.
__global__ void __launch_bounds__(PL_ONE) k_pool_grow(ba_kv_grow_args a, int shift, int most) {
    const ba_kv_pool& p = a.pool;
    __shared__ int red[PL_ONE / 64];
    __shared__ uint2 words_sh[PL_ONE];
    __shared__ int found_sh;
    const int tid = threadIdx.x, lanes = 1 << shift, l = tid & (lanes - 1), lead = (tid & 63) & ~(lanes - 1), per = PL_ONE >> shift;
    int32_t* list = p.marks + p.n_blocks;
    struct Seq {
        int len, filled, end;                                // blocks [filled, end) are those of new tokens alone
        int32_t open;                                        // the block that holds tokens and gets new ones, or -1
        bool marked;                                         // its entry is
        int32_t* row;
    };
    auto seq = [&](int s) {
        Seq r = {0, 0, 0, -1, false, nullptr};
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
        r.marked = r.open >= KV_KEPT;
        r.open = kv_block(r.open);
        if (!held(p, r.open)) r.open = -1;
        return r;
    };
    // open blocks that other lists hold too: their marks are the last sequence that is to write there, and all give them back
    auto shared = [&](int s) {                               // the one of a sequence, or -1 (before any is given back)
        const Seq r = seq(s);
        if (r.open < 0) return -1;
        const int32_t n = fresh(p.counts + r.open);
        if (n > 1) return r.open;
        if (n < 1) p.marks[r.open] = -1;                     // of no list that the pool knows: its mark may be an old one
        if (r.marked) r.row[r.len / 64] = r.open;            // the others have ended: it may be written again
        return -1;
    };
    // blocks past a list's tokens that other lists hold too are not to be written either (tokens that it has no more, and others
    // have): it gives them back and takes others.  By the counts that the call begins with, so in three passes
    auto past = [&](auto f) {
        for (int s = tid >> shift; s < a.table.n_seqs; s += per) {
            const Seq r = seq(s);
            for (int b = r.filled + l; b < r.end; b += lanes) f(r.row[b]);
        }
    };
    int any = 0;
    past([&](int32_t& e) {
        const int32_t b = kv_block(e);
        if (!held(p, b)) return;
        const int32_t n = fresh(p.counts + b);
        if (n > 1) any = 1;
        if (n > 1 || n < 1) p.marks[b] = n > 1 ? 0 : -1;
        else if (e != b) e = b;
    });
    int32_t first = shared(tid);                             // of the first PL_ONE sequences it is not looked up again
    if (__syncthreads_or(any)) {
        past([&](int32_t& e) {
            const int32_t b = kv_block(e);
            if (!held(p, b) || fresh(p.marks + b) < 0) return;
            give_back(p, b);
            e = -2 - b;                                      // wanted, and whose mark it was
        });
        __syncthreads();
        past([&](int32_t& e) {
            if (held(p, -2 - e)) p.marks[-2 - e] = -1;
        });
        __syncthreads();
        first = shared(tid);
    }
    any = 0;
    for (int s = tid; s < a.table.n_seqs; s += PL_ONE) {
        const int32_t open = s == tid ? first : shared(s);
        if (open < 0) continue;
        atomicMax(p.marks + open, s);
        any = 1;
    }
    any = __syncthreads_or(any);
    if (any) {
        if (first >= 0) atomicSub(p.counts + first, 1);
        for (int s = tid + PL_ONE; s < a.table.n_seqs; s += PL_ONE) {
            const int32_t open = seq(s).open;
            if (open >= 0 && fresh(p.marks + open) >= 0) atomicSub(p.counts + open, 1);
        }
    }
    const int free = pool_free(p, list, most, red, words_sh, &found_sh);
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
                    p.marks[block] = -1;
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
        const bool enough = base <= free;                    // all before it, and this round's, got theirs
        if (l == 0 && final && (own ? got >= 0 : enough)) p.marks[r.open] = -1;
        if (l == 0 && keeps && enough) {
            p.counts[r.open] = 1;
            if (r.marked) r.row[r.len / 64] = r.open;
        }
        if (l == 0 && got >= 0) {
            r.row[r.len / 64] = got;
            a.src[m] = r.open;
            a.dst[m] = got;
            p.counts[got] = 1;
            p.marks[got] = -1;
            atomicOr(p.used + (got >> 5), 1u << (got & 31));
        }
    }
    if (any && base > free) {                                // those that got none hold their open block as before
        auto kept = [&](auto f) {
            __syncthreads();
            for (int s = tid; s < a.table.n_seqs; s += PL_ONE) {
                const Seq r = seq(s);
                if (r.open >= 0 && fresh(p.marks + r.open) >= 0) f(r);
            }
        };
        kept([&](const Seq& r) { atomicAdd(p.counts + r.open, 1); });
        // and none of them may write there while another does not let go, not the last one either
        kept([&](const Seq& r) { r.row[r.len / 64] = fresh(p.counts + r.open) > 1 ? r.open | KV_KEPT : r.open; });
        kept([&](const Seq& r) { p.marks[r.open] = -1; });
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
__global__ void __launch_bounds__(PL_ONE) k_pool_plan(ba_kv_compact_args c) {
    const ba_kv_pool& p = c.pool;
    int32_t *src = c.src, *dst = c.dst;
    const int most = c.most;
    __shared__ int red[PL_ONE / 64];
    __shared__ uint2 words_sh[PL_ONE];
    const int tid = threadIdx.x, bit = tid & 31, words = (int)((p.n_blocks + 31) / 32), spare = (int)((int64_t)words * 32 - p.n_blocks);
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
    if (pairs)
        pool_words<true>(p, total, red, words_sh, [&](int w, uint32_t used, int before) {
            const int64_t block = (int64_t)w * 32 + bit;
            const uint32_t below = (1u << bit) - 1u;
            const bool full = used >> bit & 1u, there = block < p.n_blocks;
            const int at = full ? total - 1 - before - __popc(used & below) : w * 32 - before + __popc(~used & below);
            const bool moves = there && at < pairs;
            if (moves) (full ? src : dst)[at] = (int32_t)block;
            // the word afterwards (one store; an atomic for each of its blocks took as long as all else)
            const unsigned long long now = __ballot(!there || full != moves);
            if (bit == 0) p.used[w] = (uint32_t)(tid & 32 ? now >> 32 : now);
        });
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
        p.marks[a] = b;                                      // a is free now, b is not
        p.marks[b] = -1;
    }
    if (tid == 0) *c.n = pairs;
}

// entries of lists whose block moves: it has become free
__global__ void __launch_bounds__(PL_T) k_pool_move(ba_kv_pool p, ba_kv_table t) {
    const int64_t n = (int64_t)t.n_seqs * t.n_pages;
    for (int64_t i = (int64_t)blockIdx.x * PL_T + threadIdx.x; i < n; i += (int64_t)gridDim.x * PL_T) {
        const int64_t s = i / t.n_pages;
        int32_t* e = t.pages + s * t.stride + (i - s * t.n_pages);
        const int32_t entry = *e, b = kv_block(entry);
        if (!held(p, b) || p.counts[b] > 0) continue;
        const int32_t to = p.marks[b];
        if (held(p, to)) *e = entry < KV_KEPT ? to : to | KV_KEPT;
    }
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
    typedef uint32_t v4 __attribute__((ext_vector_type(4)));
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
            if (u < units) {                                 // not read soon: 234 MB in 42 us (5.5 TB/s; a library's copy of as many bytes 45), 49 kept in the caches
                const v4 x4 = {w[i].x, w[i].y, w[i].z, w[i].w};
                __builtin_nontemporal_store(x4, (v4*)y + u);
            }
        }
    }
}

#define POOL_TRY(call) do { const int rc_ = (call); if (rc_ != BA_OK) return rc_; } while (0)

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

static int tables_check(const ba_kv_table* tables, int n) {
    BA_REQUIRE(n >= 0 && (n == 0 || tables), "pool: bad tables");
    for (int i = 0; i < n; ++i) POOL_TRY(table_check(tables[i]));
    return BA_OK;
}

extern "C" int ba_kv_pool_count(const ba_kv_count_args* args, void* stream) {
    clear_error();
    BA_REQUIRE(args != nullptr, "null args");
    const ba_kv_pool p = args->pool;
    const ba_kv_table* tables = args->tables;
    const int n_tables = args->n_tables;
    POOL_TRY(pool_check(p));
    POOL_TRY(tables_check(tables, n_tables));
    if (p.n_blocks == 0) return BA_OK;
    hipStream_t st = (hipStream_t)stream;
    if (n_tables == 1 && p.n_blocks <= PL_FEW && (int64_t)tables[0].n_seqs * tables[0].n_pages <= 2 * PL_FEW) {
        hipLaunchKernelGGL(k_pool_count_one, dim3(1), dim3(PL_ONE), (size_t)p.n_blocks * 4, st, p, tables[0]);
        BA_LAUNCHED();
        return BA_OK;
    }
    const unsigned nb = (unsigned)((p.n_blocks + PL_T - 1) / PL_T);
    hipLaunchKernelGGL(k_pool_clear, dim3(nb), dim3(PL_T), 0, st, p);
    BA_LAUNCHED();
    for (int i = 0; i < n_tables; ++i) {
        if (tables[i].n_seqs == 0 || tables[i].n_pages == 0) continue;
        hipLaunchKernelGGL(k_pool_count, dim3(entry_grid(tables[i])), dim3(PL_T), 0, st, p, tables[i]);
        BA_LAUNCHED();
    }
    hipLaunchKernelGGL(k_pool_bits, dim3((nb + 31) / 32), dim3(PL_T), 0, st, p);
    BA_LAUNCHED();
    return BA_OK;
}

extern "C" int ba_kv_pool_free(const ba_kv_free_args* args, void* stream) {
    clear_error();
    BA_REQUIRE(args != nullptr, "null args");
    POOL_TRY(pool_check(args->pool));
    BA_REQUIRE(args->free != nullptr, "null pointer");
    hipLaunchKernelGGL(k_pool_available, dim3(1), dim3(PL_ONE), 0, (hipStream_t)stream, *args);
    BA_LAUNCHED();
    return BA_OK;
}

extern "C" int ba_kv_pool_fork(const ba_kv_fork_args* args, void* stream) {
    clear_error();
    BA_REQUIRE(args != nullptr, "null args");
    const ba_kv_fork_args& a = *args;
    POOL_TRY(pool_check(a.pool));
    POOL_TRY(table_check(a.from));
    POOL_TRY(table_check(a.to));
    BA_REQUIRE(a.n >= 0, "pool: bad sizes");
    BA_REQUIRE(a.n <= 65536, "pool: too many pairs for a call");         // each is compared with all others
    BA_REQUIRE(a.to.n_pages >= a.from.n_pages, "pool: children's lists are narrower than their parents'");
    if (a.n == 0 || a.from.n_seqs == 0 || a.to.n_seqs == 0) return BA_OK;
    BA_REQUIRE(a.parents && a.children && a.from_lengths && a.to_lengths, "null pointer");
    // (lengths of parents in another table are read while children's are written)
    BA_REQUIRE((a.from.pages == a.to.pages && a.from_lengths == a.to_lengths) || a.from_lengths + a.from.n_seqs <= a.to_lengths ||
                   a.to_lengths + a.to.n_seqs <= a.from_lengths, "pool: the children's lengths overlap the parents'");
    hipLaunchKernelGGL(k_pool_fork, dim3((unsigned)a.n), dim3(PL_T), 0, (hipStream_t)stream, a, (int)(a.from.pages == a.to.pages));
    BA_LAUNCHED();
    return BA_OK;
}

extern "C" int ba_kv_pool_trim(const ba_kv_trim_args* args, void* stream) {
    clear_error();
    BA_REQUIRE(args != nullptr, "null args");
    const ba_kv_trim_args& a = *args;
    POOL_TRY(pool_check(a.pool));
    POOL_TRY(table_check(a.table));
    BA_REQUIRE(a.n_rows >= 0 && a.n_rows < 1 << 23, "pool: bad sizes");
    const int n = a.rows ? a.n_rows : a.table.n_seqs;
    if (n == 0 || a.table.n_seqs == 0) return BA_OK;
    hipLaunchKernelGGL(k_pool_trim, dim3((unsigned)n), dim3(PL_T), 0, (hipStream_t)stream, a);
    BA_LAUNCHED();
    return BA_OK;
}

extern "C" int ba_kv_pool_grow(const ba_kv_grow_args* args, void* stream) {
    clear_error();
    BA_REQUIRE(args != nullptr, "null args");
    const ba_kv_grow_args& a = *args;
    POOL_TRY(pool_check(a.pool));
    POOL_TRY(table_check(a.table));
    BA_REQUIRE(a.max_new >= 0, "pool: bad sizes");
    BA_REQUIRE(a.n && a.missing && (a.table.n_seqs == 0 || (a.lengths && a.src && a.dst)), "null pointer");
    // blocks that a sequence may need: threads for as many, and a list of what all of them may take
    int64_t slots = ((int64_t)a.max_new + 63) / 64;
    slots = slots < a.table.n_pages ? slots : a.table.n_pages;
    int shift = 0;
    while (shift < 6 && (1 << shift) < slots) ++shift;
    const int64_t most = (slots + 1) * a.table.n_seqs;
    BA_REQUIRE(most < (int64_t)1 << 31, "pool: too many blocks for a call");     // they are counted in 32 bits
    hipLaunchKernelGGL(k_pool_grow, dim3(1), dim3(PL_ONE), 0, (hipStream_t)stream, a, shift, (int)(most < a.pool.n_blocks ? most : a.pool.n_blocks));
    BA_LAUNCHED();
    return BA_OK;
}

extern "C" int ba_kv_pool_compact(const ba_kv_compact_args* args, void* stream) {
    clear_error();
    BA_REQUIRE(args != nullptr, "null args");
    const ba_kv_compact_args& a = *args;
    POOL_TRY(pool_check(a.pool));
    POOL_TRY(tables_check(a.tables, a.n_tables));
    BA_REQUIRE(a.most >= 0 && a.most <= a.pool.n_blocks, "pool: bad sizes");
    BA_REQUIRE(a.n && (a.most == 0 || (a.src && a.dst)), "null pointer");
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(k_pool_plan, dim3(1), dim3(PL_ONE), 0, st, a);
    BA_LAUNCHED();
    for (int i = 0; i < a.n_tables && a.most; ++i) {
        if (a.tables[i].n_seqs == 0 || a.tables[i].n_pages == 0) continue;
        hipLaunchKernelGGL(k_pool_move, dim3(entry_grid(a.tables[i])), dim3(PL_T), 0, st, a.pool, a.tables[i]);
        BA_LAUNCHED();
    }
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
