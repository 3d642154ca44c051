// Log probabilities of given tokens, with the entropy of each row's distribution and its most likely classes.
//
//   z = scale * x,  lse = log sum exp(z),  p = exp(z - lse)
//   forward   logp[r] = z[r, token] - lse,  entropy[r] = -sum p log p,  the `top` classes of largest x (equal logits: the
//             lower index first) with their log probabilities
//   backward  dx[v] (+)= scale * (g [v == token] - p[v] (g + h (log p[v] + entropy))),  g = dlogp, h = dentropy
//
// Both are streams over [rows, V]: the forward pass reads the logits once, the backward pass reads them once and
// writes the gradient once; HBM bounds both.
#include "launch.hpp"
#include "row_softmax.hpp"

#include <cmath>
#include <type_traits>

namespace agrad {

namespace {

constexpr int kLpBlock = 256;
constexpr int kLpUnroll = 4;         // vectors a thread keeps in flight
constexpr uint32_t kManyRows = 1024; // more have their time by throughput, fewer by latency
constexpr uint32_t kMostHeld = 16;   // and of a row that it keeps for its alternatives
static_assert(AGRAD_MAX_TOP <= kLpBlock, "a thread an alternative");
constexpr int kLine = 8;             // vectors of a line
constexpr int kLines = 8192;         // lines that LDS holds
struct Nothing {};
constexpr int kMaxShared = 4096;     // keys that the parts of a row leave

struct LpArgs {
    const int32_t* tokens; float* logp; float* entropy; float* lse; int32_t* top_ids; float* top_logp;
    uint64_t ld; uint32_t V, top; float scale, c;
    int* err_flag;
    SharedRows shared; uint32_t parts;
};

// ---- alternatives ------------------------------------------------------------------------------------
// A class is a 64-bit key: the logit as an integer of the same order above, the complement of the index below; keys
// are distinct and descend in the order in which alternatives are given.  0 is no class.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);                   // (-0 ties with 0)
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t class_key(float x, uint32_t index) {
    return x > -INFINITY ? ((uint64_t)ordered(x) << 32) | (0xffffffffu - index) : 0ull;       // -inf and NaN: no alternative
}
__device__ __forceinline__ float key_logit(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

// What a workgroup finds.  A line is kLine neighbouring vectors (128 bytes); of each the row's one pass leaves the upper half
// of its largest logit, which is done with before the first key is written.
template <int BLOCK>
struct Candidates {
    static constexpr int kCandidates = 4 * BLOCK;    // of a row's alternatives
    static constexpr int kListed = 2 * BLOCK;        // lines with candidates
    union {
        struct {
            uint64_t key[kCandidates];
            u32x4 raw[kListed];     // vectors that hold candidates (of threads that kept theirs)
        };
        uint16_t line[BLOCK == kLpBlock ? kLines : 8];
    };
    uint32_t list[kListed];         // lines, or those vectors, that hold candidates
    uint32_t shares[BLOCK];
    uint32_t count, listed, bound;
};

// A place in a list for each lane that has something for it.  The places depend on the order in which waves arrive, the
// set does not.
__device__ __forceinline__ uint32_t take_place(uint32_t& count, bool has) {
    const uint64_t lanes = __ballot(has);
    if (lanes == 0) return 0xffffffffu;
    const uint32_t lane = threadIdx.x % kWave, first = (uint32_t)__builtin_ctzll(lanes);
    uint32_t at = 0;
    if (lane == first) at = atomicAdd(&count, (uint32_t)__popcll(lanes));
    at = (uint32_t)__builtin_amdgcn_readlane((int)at, (int)first);
    return has ? at + __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0u)) : 0xffffffffu;
}
// The same for several of a lane's, at most MOST: the first of its places.  All lanes of the wave take part.  A ballot a bit of
// MOST: a count that has more bits than are balloted would be taken for a smaller one, and lanes would share places.
template <int MOST>
__device__ __forceinline__ uint32_t take_places(uint32_t& count, uint32_t mine) {
    static_assert(MOST > 0 && MOST <= kWave, "a count of a lane");
    constexpr int BITS = 32 - __builtin_clz((unsigned)MOST);
    uint32_t before = 0, total = 0;
#pragma unroll
    for (int b = 0; b < BITS; ++b) {
        const uint64_t lanes = __ballot((mine >> b) & 1u);
        before += __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0u)) << b;
        total += (uint32_t)__popcll(lanes) << b;
    }
    if (total == 0) return 0;
    uint32_t at = 0;
    if (threadIdx.x % kWave == 0) at = atomicAdd(&count, total);
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)at) + before;
}
template <int BLOCK>
__device__ __forceinline__ void append(Candidates<BLOCK>& q, bool has, uint64_t key) {
    const uint32_t at = take_place(q.count, has);
    if (at < (uint32_t)q.kCandidates) q.key[at] = key;
}

// Keeps the largest `top` of the candidates, in descending order at the front: a key's place is the number of larger
// keys, counted (each key against all n: a tenth of the barriers of a sorting network, and faster up to some hundred
// keys, which is what a row leaves).  All threads call it after a barrier; it ends with one.
template <int BLOCK, int EACH>
__device__ __forceinline__ void prune_each(Candidates<BLOCK>& q, uint32_t n, uint32_t top) {
    uint64_t mine[EACH];
    uint32_t larger[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const uint32_t at = threadIdx.x + (uint32_t)i * BLOCK;
        mine[i] = at < n ? q.key[at] : 0ull;
        larger[i] = 0;
    }
    if (threadIdx.x / kWave * kWave < n) {                       // (waves without a key have nothing to count)
#pragma unroll 8
        for (uint32_t j = 0; j < n; ++j) {
            const uint64_t other = q.key[j];
#pragma unroll
            for (int i = 0; i < EACH; ++i) larger[i] += other > mine[i] ? 1u : 0u;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; ++i)
        if (mine[i] != 0ull && larger[i] < top) q.key[larger[i]] = mine[i];
    if (threadIdx.x == 0) q.count = n < top ? n : top;
    __syncthreads();
}
template <int BLOCK>
__device__ __forceinline__ void prune(Candidates<BLOCK>& q, uint32_t top) {
    const uint32_t n = q.count < (uint32_t)q.kCandidates ? q.count : (uint32_t)q.kCandidates;
    if (n <= (uint32_t)BLOCK) prune_each<BLOCK, 1>(q, n, top);
    else if (n <= 2u * BLOCK) prune_each<BLOCK, 2>(q, n, top);
    else prune_each<BLOCK, 4>(q, n, top);
}

// The upper half of a bound that at least `top` of the threads' values reach, as high as such a bound can be; 0 if fewer
// than `top` threads have a value (0: none).  highest: the upper half of the largest.  One wave finds it, two bits at a time,
// among the 256 halves up to the highest -- two octaves of the logit -- or, where that is not enough, bit by bit among
// all; it ends with a barrier.
template <int BLOCK>
__device__ __forceinline__ uint32_t bound_of(Candidates<BLOCK>& q, uint32_t mine, uint32_t highest, uint32_t top) {
    constexpr int EACH = BLOCK / kWave;
    q.shares[threadIdx.x] = mine;
    if (threadIdx.x == 0) q.count = q.listed = 0;
    __syncthreads();
    if (threadIdx.x < kWave) {
        uint32_t v[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) v[i] = q.shares[i * kWave + threadIdx.x] >> 16;
        auto enough = [&](uint32_t from) {
            uint32_t count = 0;
#pragma unroll
            for (int i = 0; i < EACH; ++i) count += (uint32_t)__popcll(__ballot(v[i] >= from));
            return count >= top;
        };
        uint32_t bound = highest > 0x80u + 255u ? highest - 255u : 0x80u;
        if (enough(bound)) {
#pragma unroll
            for (int bit = 6; bit >= 0; bit -= 2) {
                const uint32_t one = 1u << bit;
                const bool a = enough(bound + one), b = enough(bound + 2 * one), c = enough(bound + 3 * one);
                bound += (a ? one : 0u) + (b ? one : 0u) + (c ? one : 0u);
            }
        } else {
            bound = 0;
            for (int bit = 15; bit >= 0; --bit)
                if (enough(bound | (1u << bit))) bound |= 1u << bit;
        }
        if (threadIdx.x == 0) q.bound = bound;
    }
    __syncthreads();
    return q.bound;
}
// A logit that every class reaching the bound has at least, with few others: all that is more than -inf, for 0; next to
// zero, where the numbers below it share an upper half with -0, a little less than the bound.
__device__ __forceinline__ float bound_logit(uint32_t bound) {
    return bound == 0 ? -3.4028234663852886e38f : bound == 0x8000u ? -1.2e-38f : key_logit((uint64_t)bound << 48);
}
// the order of the upper halves of fp32 numbers (-0 with 0)
__device__ __forceinline__ uint32_t ordered_half(uint32_t h) { return (h & 0x8000u) && h != 0x8000u ? ~h & 0xffffu : h | 0x8000u; }

// The largest of n keys, one a thread and step: right whatever they are, and slow.
template <int BLOCK, typename KeyAt>
__device__ __forceinline__ void top_by_steps(uint32_t n, uint32_t top, Candidates<BLOCK>& q, KeyAt key_at) {
    if (threadIdx.x == 0) q.count = 0;
    __syncthreads();
    uint64_t floor_key = 0;
    for (uint32_t i0 = 0; i0 < n; i0 += BLOCK) {
        const uint32_t i = i0 + threadIdx.x;
        const uint64_t key = i < n ? key_at(i) : 0ull;
        append(q, key > floor_key, key);
        __syncthreads();
        const bool full = q.count > (uint32_t)(q.kCandidates - BLOCK);
        __syncthreads();
        if (full) {
            prune<BLOCK>(q, top);
            floor_key = q.count == top ? q.key[top - 1] : 0ull;
            __syncthreads();
        }
    }
    prune<BLOCK>(q, top);
}

// The alternatives of a stretch of a row's vectors (the first stretch: and of the elements outside the vectors) of which
// every thread has seen its share, the vectors whose number is its own modulo BLOCK, and kept the largest logit, `best`.
// At least `top` classes reach the top-th largest of those BLOCK values, and hardly more do (75 of 151936 for top = 64,
// 180 for top = 128, as the shares are interleaved).  With them known, the row is not read again but for the lines whose
// largest logit reaches the bound -- or not at all, where the threads still hold their vectors (HELD; tops: their largest
// logits).  (Reading the shares again instead of lines reads the whole row: eight threads have a part in each 128 bytes.
// 8192 rows of 128256 bf16, top 64: 595 us.)  A row whose largest logits are equal in great number, share the upper half of their
// bits, or crowd into few shares, can leave more than LDS holds and goes the slow way: all equal, those rows take 1830 us for 344;
// fp32 rows about 1000, where an upper half is a step of 4, 750 for 131 (4096 of 50257, top 20); the worst found, such rows in
// ascending order, 12000.
template <typename T, int VEC, int BLOCK, bool HELD, int U>
__device__ __forceinline__ void row_top(const T* base, const RowParts<T, VEC>& parts, const Stretch& part, uint32_t top, float best, float largest,
                                        const typename RawVec<T, VEC>::type (&held)[U], const float (&tops)[U],
                                        uint32_t skew, Candidates<BLOCK>& q) {
    typedef RawVec<T, VEC> Raw;
    const uint32_t extra = part.lo == 0 ? parts.extra : 0u, vectors = part.hi - part.lo;
    const uint32_t bound = bound_of<BLOCK>(q, (uint32_t)(class_key(best, 0u) >> 32), ordered(largest) >> 16, top);
    const float least = bound_logit(bound);
    const T* body = base + parts.head;
    bool fits = true;
    auto append_vector = [&](bool has, uint32_t number, const typename Raw::type& raw) {
        float v[VEC];
        Raw::unpack(raw, v);
        uint32_t mine = 0;
#pragma unroll
        for (int k = 0; k < VEC; ++k) mine += has && v[k] >= least ? 1u : 0u;
        uint32_t at = take_places<VEC>(q.count, mine);
        if (mine == 0) return;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            if (!(v[k] >= least)) continue;
            if (at < (uint32_t)q.kCandidates) q.key[at] = class_key(v[k], parts.head + number * VEC + k);
            ++at;
        }
    };
    if constexpr (HELD) {
        // first whole vectors, then classes, an element a thread: a place for each class of four vectors costs more
        uint32_t reach = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) reach += tops[u] >= least ? 1u : 0u;
        uint32_t at = take_places<U>(q.listed, reach);            // (all U vectors of a thread may reach it)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!(tops[u] >= least)) continue;
            if (at < (uint32_t)q.kListed) {
                reinterpret_cast<typename Raw::type*>(q.raw)[at] = held[u];
                q.list[at] = part.lo + u * BLOCK + threadIdx.x;
            }
            ++at;
        }
        __syncthreads();
        const uint32_t n = q.listed;
        fits = n <= (uint32_t)q.kListed;
        const uint32_t classes = fits ? n * VEC : 0u;
        for (uint32_t i = threadIdx.x; i / kWave * kWave < classes; i += BLOCK) {
            float v[1];
            RawVec<T, 1>::unpack(reinterpret_cast<const T*>(q.raw)[i < classes ? i : 0u], v);
            append(q, i < classes && v[0] >= least, class_key(v[0], parts.head + q.list[i < classes ? i / VEC : 0u] * VEC + i % VEC));
        }
    } else {
        const uint32_t all_lines = (vectors + skew + kLine - 1) / kLine, lines = all_lines <= (uint32_t)kLines ? all_lines : 0u;
        const uint32_t from = bound < 0x80u ? 0x80u : bound;                 // (-inf is 0x7f)
        constexpr int EACH = 8;                                              // lines a thread looks at: one load
        for (uint32_t j0 = 0; j0 < lines; j0 += BLOCK * EACH) {
            const uint32_t j = j0 + threadIdx.x * EACH;
            u32x4 w = *reinterpret_cast<const u32x4*>(q.line + (j < lines ? j : 0u));
            const uint32_t pair[4] = {w.x, w.y, w.z, w.w};
            uint32_t reach = 0;
#pragma unroll
            for (int k = 0; k < EACH; ++k) {
                const uint32_t h = k % 2 ? pair[k / 2] >> 16 : pair[k / 2] & 0xffffu;
                if (j + k < lines && ordered_half(h) >= from) reach |= 1u << k;
            }
            uint32_t at = take_places<EACH>(q.listed, (uint32_t)__popc(reach));
            for (; reach != 0; reach &= reach - 1u, ++at)
                if (at < (uint32_t)q.kListed) q.list[at] = j + (uint32_t)__builtin_ctz(reach);
        }
        __syncthreads();
        const uint32_t n = q.listed;
        fits = n <= (uint32_t)q.kListed && lines == all_lines;
        const uint32_t again = fits ? n * kLine : 0u;
        constexpr int AHEAD = 2;
        for (uint32_t i0 = threadIdx.x; i0 / kWave * kWave < again; i0 += BLOCK * AHEAD) {
            typename Raw::type raw[AHEAD];
            uint32_t number[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const uint32_t i = i0 + u * BLOCK;
                number[u] = i < again ? q.list[i / kLine] * kLine + i % kLine - skew : vectors;      // (before the first: large)
                raw[u] = Raw::load(body + (uint64_t)(part.lo + (number[u] < vectors ? number[u] : 0u)) * VEC);
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) append_vector(number[u] < vectors, part.lo + number[u], raw[u]);
        }
    }
    if (threadIdx.x < extra) {
        const uint32_t e = parts.extra_at(threadIdx.x);
        float x[1];
        VecIO<T, 1>::load(base + e, x);
        append(q, x[0] >= least, class_key(x[0], e));
    }
    __syncthreads();
    if (!fits || q.count > (uint32_t)q.kCandidates) {
        __syncthreads();
        const uint32_t in_vectors = vectors * VEC;
        top_by_steps<BLOCK>(in_vectors + extra, top, q, [&](uint32_t i) {
            const uint32_t e = i < in_vectors ? parts.head + part.lo * VEC + i : parts.extra_at(i - in_vectors);
            float x[1];
            VecIO<T, 1>::load(base + e, x);
            return class_key(x[0], e);
        });
    } else {
        prune<BLOCK>(q, top);
    }
}

// The `top` largest of the n keys that a row's parts left, descending: key k of part j is at k * parts + j, so that the
// parts' first keys, among which the row's largest are, fall to different threads.
struct KeyList {
    uint64_t key[kMaxShared / kLpBlock];          // a thread's share
    __device__ __forceinline__ KeyList(const unsigned long long* keys, uint32_t n) {
#pragma unroll
        for (int i = 0; i < kMaxShared / kLpBlock; ++i) {
            const uint32_t at = threadIdx.x + i * kLpBlock;
            key[i] = 0;
            if (i * (uint32_t)kLpBlock < n) key[i] = get_shared(keys + (at < n ? at : 0u));
            if (at >= n) key[i] = 0;
        }
    }
};
template <int BLOCK>
__device__ __forceinline__ void join_tops(const KeyList& mine, const unsigned long long* keys, uint32_t n, uint32_t top, float largest, Candidates<BLOCK>& q) {
    constexpr int EACH = kMaxShared / BLOCK;
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) best = max(best, (uint32_t)(mine.key[i] >> 32));
    const uint32_t bound = bound_of<BLOCK>(q, best, ordered(largest) >> 16, top);
#pragma unroll
    for (int i = 0; i < EACH; ++i)
        if (i * (uint32_t)BLOCK < n) append(q, mine.key[i] != 0ull && (uint32_t)(mine.key[i] >> 48) >= bound, mine.key[i]);
    __syncthreads();
    if (q.count > (uint32_t)q.kCandidates) {
        __syncthreads();
        top_by_steps<BLOCK>(n, top, q, [&](uint32_t i) { return (uint64_t)get_shared(keys + i); });
    } else {
        prune<BLOCK>(q, top);
    }
}

// ---- forward -----------------------------------------------------------------------------------------
// A workgroup reads a row, or a part of it, once, U vectors a thread in flight.  With HELD the part is no longer than those, and
// they stay in registers for the alternatives; with LINES the pass leaves every line's largest logit for them.  HBM bounds long
// batches (4096 rows of 50257 fp32 with entropy 126 us, 6.5 TB/s; 8192 rows of 128256 bf16 with 64 alternatives 346 us, 6.1 TB/s),
// latency the small ones (one row of 128256 bf16 with 20 alternatives 9.5 us, 5.5 without).
enum LpMode { PLAIN, LINES, HELD };
template <typename T, int VEC, bool ENT, LpMode MODE, int BLOCK, int U>
__global__ void __launch_bounds__(BLOCK)
logprobs_fwd_kernel(const T* __restrict__ x, const LpArgs a) {
    __shared__ RowStat lds[BLOCK / kWave];
    __shared__ std::conditional_t<MODE == PLAIN, Nothing, Candidates<BLOCK>> found;
    __shared__ uint32_t word;
    typedef RawVec<T, VEC> Raw;
    const uint32_t row = blockIdx.x / a.parts, nth = blockIdx.x - row * a.parts;
    const T* base = x + row * a.ld;
    const RowParts<T, VEC> parts(base, a.V);
    const Stretch part(parts.nvec, nth, a.parts);
    const T* body = base + parts.head;
    typename Raw::type raw[U];
    float tops[U];
    RowStat t = empty_stat();
    // lane 0 of the part's first wave stands before its first vector, where that is not at 128 bytes: whole lines a wave
    const uint32_t length = part.hi - part.lo, skew = MODE == HELD ? 0u : line_skew<VEC>(body + (uint64_t)part.lo * VEC, length, BLOCK * U);
    auto inside = [&](uint32_t i) { return MODE == HELD ? i < part.hi : i - part.lo < length; };
    auto read = [&](uint32_t i0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t i = i0 + u * BLOCK;
            raw[u] = Raw::load(body + (uint64_t)(inside(i) ? i : part.lo) * VEC);
        }
    };
    auto absorb = [&](uint32_t i0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            tops[u] = -INFINITY;
            if (inside(i0 + u * BLOCK)) {
                float v[VEC];
                Raw::unpack(raw[u], v);
                tops[u] = absorb_stat<ENT, VEC>(t, v, a.c);
            }
        }
    };
    if (MODE == HELD && part.lo < part.hi) read(part.lo + threadIdx.x);
    // the token's logit, and the elements outside the vectors
    const int32_t token = a.tokens != nullptr ? a.tokens[row] : -1;
    const bool asked = token >= 0 && (uint32_t)token < a.V;
    float at[1];
    VecIO<T, 1>::load(base + (asked ? token : 0), at);
    if (nth == 0 && threadIdx.x < parts.extra) {
        float v[1];
        VecIO<T, 1>::load(base + parts.extra_at(threadIdx.x), v);
        absorb_stat<ENT, 1>(t, v, a.c);
    }
    if constexpr (MODE == HELD) {
        absorb(part.lo + threadIdx.x);
    } else {
        const uint32_t lane = threadIdx.x % kWave;
        const uint32_t first = part.lo - skew + lane;                                 // (of wave 0; whole waves)
        for (uint32_t i0 = threadIdx.x - lane; i0 < length + skew; i0 += BLOCK * U) {
            read(first + i0);
            absorb(first + i0);
            if constexpr (MODE == LINES) {
                static_assert(kLine == 8, "the lanes of half a DPP row");
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float m = fmaxf(tops[u], dpp_move<kDppQuadXor1>(tops[u]));
                    m = fmaxf(m, dpp_move<kDppQuadXor2>(m));
                    m = fmaxf(m, dpp_move<kDppRowHalfMirror>(m));
                    const uint32_t line = (i0 + u * BLOCK + lane) / kLine;
                    if (lane % kLine == 0 && line < (uint32_t)kLines) found.line[line] = (uint16_t)(__float_as_uint(m) >> 16);
                }
            }
        }
    }
    const float best = t.m;
    t = block_stat<BLOCK, ENT>(t, a.c, lds);
    if constexpr (MODE != PLAIN)
        if (a.top != 0) row_top<T, VEC, BLOCK, MODE == HELD, U>(base, parts, part, a.top, best, t.m, raw, tops, skew, found);
    if constexpr (BLOCK == kLpBlock) if (a.parts > 1) {
        if (threadIdx.x == 0) {
            float* to = a.shared.stats + 4 * (uint64_t)blockIdx.x;
            put_shared(to, t.m);
            put_shared(to + 1, t.s);
            if (ENT) put_shared(to + 2, t.d);
        }
        unsigned long long* keys = a.shared.keys + (uint64_t)row * a.parts * a.top;
        if constexpr (MODE != PLAIN)
            if (threadIdx.x < a.top)
                put_shared(keys + threadIdx.x * a.parts + nth, (unsigned long long)(threadIdx.x < found.count ? found.key[threadIdx.x] : 0ull));
        if (!workgroup_arrives_last(a.shared.tickets + row, a.parts, &word)) return;
        t = empty_stat();
        if (threadIdx.x < a.parts) {
            const float* from = a.shared.stats + 4 * ((uint64_t)row * a.parts + threadIdx.x);
            t = RowStat{get_shared(from), get_shared(from + 1), ENT ? get_shared(from + 2) : 0.0f};
        }
        if constexpr (MODE != PLAIN) {
            const KeyList mine(keys, a.parts * a.top);                // (asked for before the statistics are put together)
            t = block_stat<BLOCK, ENT>(t, a.c, lds);
            if (a.top != 0) join_tops<BLOCK>(mine, keys, a.parts * a.top, a.top, t.m, found);
        } else {
            t = block_stat<BLOCK, ENT>(t, a.c, lds);
        }
    }
    const bool empty = t.m == -INFINITY && t.s == 0.0f;
    const float log_s = logf(t.s);                                // -inf for an empty row
    if (threadIdx.x == 0) {
        if (a.lse != nullptr) a.lse[row] = empty ? -INFINITY : t.m * a.scale + log_s;
        if (ENT) a.entropy[row] = empty ? 0.0f : log_s - kLn2 * (t.d / t.s);
        if (a.tokens != nullptr) {
            if (!asked && token != -1) *a.err_flag = 1;
            a.logp[row] = asked && !empty ? (at[0] - t.m) * a.scale - log_s : 0.0f;
        }
    }
    if constexpr (MODE != PLAIN) {
        if (threadIdx.x >= a.top) return;
        const bool there = threadIdx.x < found.count;
        const uint64_t key = there ? found.key[threadIdx.x] : 0ull;
        const uint64_t to = (uint64_t)row * a.top + threadIdx.x;
        a.top_ids[to] = there ? (int32_t)key_index(key) : -1;
        a.top_logp[to] = there ? (key_logit(key) - t.m) * a.scale - log_s : -INFINITY;
    }
}

// ---- backward ----------------------------------------------------------------------------------------
// One vector a thread, a workgroup a chunk of a row (the most independent waves: a stream of one read and one write runs
// best that way here: 4096 rows of 128256 fp32 687 us, 2048 rows of 50257 bf16 66 us, 6.1 and 6.3 TB/s).  With l = log p:
// dx = scale * (g [v == token] - p (g + h entropy + h l)).
struct LpBwdArgs {
    const int32_t* tokens; const float* lse; const float* entropy; const float* dlogp; const float* dentropy;
    uint64_t ld; uint32_t V; float scale; uint32_t accumulate;
    int* err_flag;
};

struct LpRow {
    float scale, lse, a, h, g;          // a = scale * (g + h * entropy), h, g already multiplied by scale
    uint32_t token;
};

__device__ __forceinline__ float lp_grad(float x, const LpRow& r, uint32_t e) {
    const float l = x * r.scale - r.lse;
    const float p = __builtin_amdgcn_exp2f(l * kLog2eHi);
    float d = -p * __builtin_fmaf(r.h, fmaxf(l, -200.0f), r.a);
    if (e == r.token) d = d + r.g;
    return d;
}

template <typename T, int VEC>
__device__ __forceinline__ void lp_store(T* to, float (&d)[VEC], uint32_t accumulate) {
    if (accumulate) {
        float old[VEC];
        VecIO<T, VEC>::load(to, old);
#pragma unroll
        for (int k = 0; k < VEC; ++k) d[k] = old[k] + d[k];
    }
    store_grad<T, VEC>(to, d);
}

// A row whose lse is so large that fp32 holds little of the logarithm beside the offset (all classes at a mask's lowest value:
// nothing of it, p would be 1 each; with a scale above 1 the lse is -inf like that of a row without classes).  The row's
// first workgroup takes all of it and sums it up again about its largest logit; it has read the row before it writes, so dx
// may be x here too.  Reading twice costs many rows a factor of two (4096 of 128256 fp32 1423 us for 684, 2048 of 50257 bf16 141 for
// 64), a workgroup a row a few long ones more (one row of 151936 bf16 52 us for 4, 256 rows 135 for 26).
constexpr float kLargeLse = 256.0f;          // (an error of 2^-17 in log p)
template <typename T, int VEC, int BLOCK>
__device__ void lp_bwd_row(const T* base, T* out, const RowParts<T, VEC>& parts, LpRow r, uint32_t accumulate) {
    __shared__ RowStat lds[BLOCK / kWave];
    const float c = r.scale * kLog2eHi;
    RowStat t = empty_stat();
    float e[1] = {-INFINITY};
    if (threadIdx.x < parts.extra) VecIO<T, 1>::load(base + parts.extra_at(threadIdx.x), e);
    absorb_stat<false, 1>(t, e, c);
    for (uint32_t i = threadIdx.x; i < parts.nvec; i += BLOCK) {
        float v[VEC];
        VecIO<T, VEC>::load(base + parts.head + (uint64_t)i * VEC, v);
        absorb_stat<false, VEC>(t, v, c);
    }
    t = block_stat<BLOCK, false>(t, c, lds);
    r.lse = logf(t.s);
    if (t.m == -INFINITY && t.s == 0.0f) {                 // no class: no gradient
        t.m = 0.0f;
        r.lse = INFINITY;
        r.a = r.h = r.g = 0.0f;
    }
    if (threadIdx.x < parts.extra) {
        const uint32_t at = parts.extra_at(threadIdx.x);
        e[0] = lp_grad(e[0] - t.m, r, at);
        lp_store<T, 1>(out + at, e, accumulate);
    }
    for (uint32_t i = threadIdx.x; i < parts.nvec; i += BLOCK) {
        const uint32_t first = parts.head + i * VEC;
        float v[VEC];
        VecIO<T, VEC>::load(base + first, v);
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = lp_grad(v[k] - t.m, r, first + k);
        lp_store<T, VEC>(out + first, v, accumulate);
    }
}

template <typename T, int VEC, int BLOCK>
__global__ void __launch_bounds__(BLOCK)
logprobs_bwd_kernel(const T* x, T* dx, const LpBwdArgs a, const FastDiv32 chunks) {
    const uint32_t row = chunks.div(blockIdx.x), chunk = blockIdx.x - row * chunks.d;
    const T* base = x + (uint64_t)row * a.ld;
    T* out = dx + (uint64_t)row * a.ld;
    LpRow r;
    const int32_t token = a.tokens != nullptr ? a.tokens[row] : -1;
    const bool asked = token >= 0 && (uint32_t)token < a.V;
    if (!asked && token != -1 && chunk == 0 && threadIdx.x == 0) *a.err_flag = 1;
    r.scale = a.scale;
    r.lse = a.lse[row];
    r.token = asked ? (uint32_t)token : 0xffffffffu;
    r.g = asked && a.dlogp != nullptr ? a.scale * a.dlogp[row] : 0.0f;
    r.h = a.dentropy != nullptr ? a.scale * a.dentropy[row] : 0.0f;
    r.a = a.dentropy != nullptr ? __builtin_fmaf(r.h, a.entropy[row], r.g) : r.g;
    const RowParts<T, VEC> parts(base, a.V);
    if (fabsf(r.lse) > kLargeLse) {
        if (chunk == 0) lp_bwd_row<T, VEC, BLOCK>(base, out, parts, r, a.accumulate);
        return;
    }
    if (chunk == 0 && threadIdx.x < parts.extra) {
        const uint32_t e = parts.extra_at(threadIdx.x);
        float v[1];
        VecIO<T, 1>::load(base + e, v);
        v[0] = lp_grad(v[0], r, e);
        lp_store<T, 1>(out + e, v, a.accumulate);
    }
    const uint32_t i = chunk * BLOCK + threadIdx.x - line_skew<VEC>(base + parts.head);
    if (i >= parts.nvec) return;
    const uint32_t first = parts.head + i * VEC;
    float v[VEC];
    VecIO<T, VEC>::load(base + first, v);
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = lp_grad(v[k], r, first + k);
    lp_store<T, VEC>(out + first, v, a.accumulate);
}

template <typename T, int VEC, LpMode MODE, int BLOCK = kLpBlock, int U = kLpUnroll>
void lp_fwd_launch(hipStream_t s, const T* x, const LpArgs& a, uint64_t rows) {
    const dim3 grid((uint32_t)rows * a.parts), block(BLOCK);
    if (a.entropy) hipLaunchKernelGGL((logprobs_fwd_kernel<T, VEC, true, MODE, BLOCK, U>), grid, block, 0, s, x, a);
    else hipLaunchKernelGGL((logprobs_fwd_kernel<T, VEC, false, MODE, BLOCK, U>), grid, block, 0, s, x, a);
}

// Rows of up to kLpUnroll vectors a thread, in the smallest workgroup that holds one: with many rows the reductions of its waves
// are most of the time (32768 rows of 257 fp32 in 64 threads and in 256: 15 and 40 us without alternatives, 26 and 87 with 5).
// The alternatives need some threads each, for a useful bound: two do where there are many rows (32768 rows of 2000 bf16, 64
// alternatives: 82 us, with four 127), and cost a few rows their latency (512 rows: 8.0 us, with four 7.2).
template <typename T, int VEC>
int lp_fwd_short(hipStream_t s, const T* x, const LpArgs& a, uint64_t rows) {
    const uint32_t vectors = a.V / VEC, each = rows > kManyRows ? 2 : 4;
    auto fits = [&](uint32_t block) { return vectors <= block * kLpUnroll && each * a.top <= block; };
    if (a.top == 0 && fits(64)) lp_fwd_launch<T, VEC, PLAIN, 64>(s, x, a, rows);
    else if (a.top == 0 && fits(128)) lp_fwd_launch<T, VEC, PLAIN, 128>(s, x, a, rows);
    else if (fits(64)) lp_fwd_launch<T, VEC, HELD, 64>(s, x, a, rows);
    else if (fits(128)) lp_fwd_launch<T, VEC, HELD, 128>(s, x, a, rows);
    else lp_fwd_launch<T, VEC, HELD>(s, x, a, rows);
    return check_hip(hipGetLastError(), "token log probabilities launch");
}

template <typename T>
int lp_fwd_typed(hipStream_t s, const T* x, LpArgs a, uint64_t rows) {
    constexpr int WIDE = WideVec<T>::value;
    const uint32_t vectors = a.V / WIDE;
    // Short rows with many alternatives go by single elements: of fewer vectors than one and a half times the alternatives the threads'
    // largest logits give no useful bound (1000 bf16 classes, 128 alternatives: 28.6 us, all of them candidates; by elements 6.9).
    // Up to twice as many vectors, elements are faster for a few rows (512 rows of 600 bf16, 50 alternatives 6.2 against 6.9 us) and
    // vectors for many (32768 rows 69 against 105).
    const bool many = a.V <= (uint32_t)kLpBlock * kLpUnroll && 2 * vectors < (rows > kManyRows ? 3 : 4) * a.top;
    if (a.V < 4 * WIDE || many) return lp_fwd_short<T, 1>(s, x, a, rows);
    if (vectors <= (uint32_t)kLpBlock / 2 * kLpUnroll) return lp_fwd_short<T, WIDE>(s, x, a, rows);
    // (with alternatives a row is shared from where a workgroup cannot hold it: 4096 vectors in one, one row 8.4 us, 256 rows 9.6; in
    // four parts 9.5 and 13.2)
    a.parts = a.top != 0 && vectors <= kLpBlock * kMostHeld ? 1u : row_parts(rows, vectors);
    uint64_t slab = rows;
    if (a.top != 0) {
        if (a.parts * a.top > (uint32_t)kMaxShared) a.parts = kMaxShared / a.top;
        // a part's lines have to fit LDS: rows of more than kLines lines are cut, so many rows a launch as the parts' memory takes
        const uint32_t least = (vectors + kLine) / (uint32_t)(kLines * kLine) + 1;
        if (least > a.parts) {
            a.parts = least < kMaxShared / a.top ? least : kMaxShared / a.top;
            if (a.parts > kMaxParts) a.parts = kMaxParts;
            slab = kSharedParts / a.parts;
        }
    }
    const uint32_t longest = (vectors + a.parts - 1) / a.parts;
    // (held against read again by lines: 8192 rows of 8192 fp32 with 20 alternatives 45.7 against 60.3 us, of 16384 88 against 94)
    auto held = [&](uint32_t each) { return a.top != 0 && longest <= kLpBlock * each; };
    for (uint64_t r0 = 0; r0 < rows; r0 += slab) {
        const uint64_t n = rows - r0 < slab ? rows - r0 : slab;
        LpArgs b = a;
        if (b.tokens) { b.tokens += r0; b.logp += r0; }
        if (b.entropy) b.entropy += r0;
        if (b.lse) b.lse += r0;
        if (b.top) { b.top_ids += r0 * b.top; b.top_logp += r0 * b.top; }
        const T* from = x + r0 * a.ld;
        if (held(4)) lp_fwd_launch<T, WIDE, HELD, kLpBlock, 4>(s, from, b, n);
        else if (held(8)) lp_fwd_launch<T, WIDE, HELD, kLpBlock, 8>(s, from, b, n);
        else if (held(kMostHeld)) lp_fwd_launch<T, WIDE, HELD, kLpBlock, kMostHeld>(s, from, b, n);
        else if (a.top != 0) lp_fwd_launch<T, WIDE, LINES>(s, from, b, n);
        else lp_fwd_launch<T, WIDE, PLAIN>(s, from, b, n);
    }
    return check_hip(hipGetLastError(), "token log probabilities launch");
}

template <typename T>
int lp_bwd_typed(hipStream_t s, const T* x, T* dx, LpBwdArgs a, uint64_t rows) {
    constexpr int WIDE = WideVec<T>::value;
    // rows are realigned by their first elements, which needs both tensors at one offset within 16 bytes
    const bool wide = a.V >= 4 * WIDE && ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15u) == 0;
    const uint32_t vec = wide ? WIDE : 1;
    // (short rows leave most of a larger workgroup's threads idle: 32768 rows of 257 fp32 16.4 against 24.8 us, of 2048 bf16 42.5
    // against 45.0; longer rows are the same in both)
    const uint32_t block = a.V / vec <= 256u ? 64u : kLpBlock;
    const bool lines = ((reinterpret_cast<uintptr_t>(x) | (rows > 1 ? a.ld * sizeof(T) : 0u)) & 127u) == 0;      // every row at 128 bytes
    const uint32_t chunks = (a.V / vec + (wide && !lines ? 7u : 0u) + block - 1) / block;
    uint64_t max_rows = 0x00ffffffull / chunks;                  // workgroups of a launch: 2^32 threads
    if (max_rows == 0) max_rows = 1;
    for (uint64_t r0 = 0; r0 < rows; r0 += max_rows) {
        const uint64_t n = rows - r0 < max_rows ? rows - r0 : max_rows;
        LpBwdArgs b = a;
        if (b.tokens) b.tokens += r0;
        b.lse += r0;
        if (b.entropy) b.entropy += r0;
        if (b.dlogp) b.dlogp += r0;
        if (b.dentropy) b.dentropy += r0;
        const dim3 grid((uint32_t)(n * chunks));
#define AGRAD_LP(VEC, BLOCK) hipLaunchKernelGGL((logprobs_bwd_kernel<T, VEC, BLOCK>), grid, dim3(BLOCK), 0, s, x + r0 * a.ld, dx + r0 * a.ld, b, FastDiv32(chunks))
        if (wide && block == 64) AGRAD_LP(WIDE, 64);
        else if (wide) AGRAD_LP(WIDE, kLpBlock);
        else if (block == 64) AGRAD_LP(1, 64);
        else AGRAD_LP(1, kLpBlock);
#undef AGRAD_LP
    }
    return check_hip(hipGetLastError(), "token log probabilities backward launch");
}

}  // namespace

uint64_t shared_rows_bytes() { return kSharedRowsBytes; }

SharedRows shared_rows(void* scratch) {
    char* at = static_cast<char*>(scratch);
    return SharedRows{reinterpret_cast<float*>(at), reinterpret_cast<unsigned long long*>(at + 16ull * kSharedParts),
                      reinterpret_cast<uint32_t*>(at + (16ull + 8ull * AGRAD_MAX_TOP) * kSharedParts),
                      reinterpret_cast<float*>(at + (16ull + 8ull * AGRAD_MAX_TOP + 4ull) * kSharedParts)};
}

// Parts of a row: of 1024 vectors, four a thread, or 2048 where that makes 256 workgroups of all rows, but not more than 512
// workgroups, or 1024 where the parts stay longer than 4096 vectors (a part costs its workgroup's reductions, and the parts
// are put together one after the other).  Up to 2048 vectors one workgroup is as fast: what one leaves for another takes 2 us to
// arrive.  One row of 2048 vectors 4.1 us (two parts 4.9), of 4096 5.5 (four parts 4.9), of 16384 18.3 (four parts 7.3, eight 5.7,
// sixteen 5.2); 64 rows of 8192 without alternatives: two parts 9.4, four 7.7, eight 7.7, sixteen 10.5; 37 rows of 12564 with
// 5: five parts 12.6, seven 11.7, thirteen 12.4, nineteen 14.3; 48 rows of 18992 with 8: five parts 14.5, ten 14.2, nineteen 15.9.
uint32_t row_parts(uint64_t rows, uint32_t vectors) {
    if (vectors <= 2048u) return 1u;
    uint64_t parts = (vectors + 1023u) / 1024u;
    if (parts * rows >= 256) parts = (vectors + 2047u) / 2048u;
    uint64_t most = 512 / rows;
    if (most == 0 || vectors / most > 4096) most = kSharedParts / rows;
    if (parts > most) parts = most;
    if (parts > kMaxParts) parts = kMaxParts;
    return parts < 1 ? 1u : (uint32_t)parts;
}

int logits_check(const char* what, int dtype, const void* x, const void* dx, uint64_t rows, uint32_t V, uint64_t ld, float scale) {
    if (dtype != AGRAD_F32 && dtype != AGRAD_BF16) return set_error(AGRAD_EINVAL, "%s: unknown dtype %d", what, dtype);
    if (V == 0 || V >= 0x7fffffffu) return set_error(AGRAD_EINVAL, "%s: %u classes", what, V);
    if (ld < V || ld > 0xffffffffull) return set_error(AGRAD_EINVAL, "%s: row stride %llu for %u classes", what, (unsigned long long)ld, V);
    // (a launch has fewer than 2^32 threads; the largest workgroup here has 1024)
    if (rows >= 0x00400000ull) return set_error(AGRAD_EINVAL, "%s: at most %u rows a call", what, 0x003fffffu);
    // (above 2e38 the product with log2(e), by which the kernels take distances, is not finite: a distance of 0 would be NaN)
    if (!(scale > 0.0f) || !(scale <= 2e38f)) return set_error(AGRAD_EINVAL, "%s: the scale must be positive and at most 2e38", what);
    const uintptr_t es = dtype_size(dtype);
    if (reinterpret_cast<uintptr_t>(x) % es || reinterpret_cast<uintptr_t>(dx) % es)
        return set_error(AGRAD_EINVAL, "%s: logits or gradient not aligned to their elements", what);
    return AGRAD_OK;
}

int launch_logprobs_fwd(hipStream_t s, int dtype, const void* logits, const int32_t* tokens, float* logp, float* entropy,
                        float* lse, int32_t* top_ids, float* top_logp, uint64_t rows, uint32_t V, uint64_t ld, uint32_t top,
                        float scale, int* err_flag, void* scratch) {
    const char* what = "token log probabilities";
    if (int rc = logits_check(what, dtype, logits, nullptr, rows, V, ld, scale)) return rc;
    if (top > AGRAD_MAX_TOP) return set_error(AGRAD_EINVAL, "%s: at most %u alternatives, got %u", what, AGRAD_MAX_TOP, top);
    if (rows == 0) return AGRAD_OK;
    if (logits == nullptr) return set_error(AGRAD_EINVAL, "%s: null logits", what);
    if ((tokens != nullptr) != (logp != nullptr)) return set_error(AGRAD_EINVAL, "%s: tokens and logp go together", what);
    if ((top != 0) != (top_ids != nullptr) || (top != 0) != (top_logp != nullptr))
        return set_error(AGRAD_EINVAL, "%s: top_ids and top_logp are given exactly when top > 0", what);
    if (logp == nullptr && entropy == nullptr && lse == nullptr && top == 0) return set_error(AGRAD_EINVAL, "%s: nothing to compute", what);
    const float c = (float)((double)scale * 1.4426950408889634);
    const LpArgs a{tokens, logp, entropy, lse, top_ids, top_logp, ld, V, top, scale, c, err_flag, shared_rows(scratch), 1u};
    if (dtype == AGRAD_F32) return lp_fwd_typed<float>(s, (const float*)logits, a, rows);
    return lp_fwd_typed<bf16_t>(s, (const bf16_t*)logits, a, rows);
}

int launch_logprobs_bwd(hipStream_t s, int dtype, const void* logits, const int32_t* tokens, const float* lse,
                        const float* entropy, const float* dlogp, const float* dentropy, void* dlogits, uint64_t rows,
                        uint32_t V, uint64_t ld, float scale, uint32_t flags, int* err_flag) {
    const char* what = "token log probabilities backward";
    if (int rc = logits_check(what, dtype, logits, dlogits, rows, V, ld, scale)) return rc;
    if (flags & ~(uint32_t)AGRAD_ACC_INPUT_GRAD) return set_error(AGRAD_EINVAL, "%s: unknown flag bits 0x%x", what, flags);
    if (rows == 0) return AGRAD_OK;
    if (logits == nullptr || dlogits == nullptr || lse == nullptr) return set_error(AGRAD_EINVAL, "%s: null operand", what);
    if (dlogp == nullptr && dentropy == nullptr) return set_error(AGRAD_EINVAL, "%s: neither dlogp nor dentropy", what);
    if (dlogp != nullptr && tokens == nullptr) return set_error(AGRAD_EINVAL, "%s: dlogp without tokens", what);
    if (dentropy != nullptr && entropy == nullptr) return set_error(AGRAD_EINVAL, "%s: dentropy without the entropy", what);
    const LpBwdArgs a{dlogp != nullptr ? tokens : nullptr, lse, entropy, dlogp, dentropy, ld, V, scale,
                      (flags & AGRAD_ACC_INPUT_GRAD) ? 1u : 0u, err_flag};
    if (dtype == AGRAD_F32) return lp_bwd_typed<float>(s, (const float*)logits, (float*)dlogits, a, rows);
    return lp_bwd_typed<bf16_t>(s, (const bf16_t*)logits, (bf16_t*)dlogits, a, rows);
}

}  // namespace agrad
