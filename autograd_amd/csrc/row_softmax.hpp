// Device parts shared by the operators that read rows of logits (logprobs.hip, distill.hip): the statistics of a
// softmax over scale * x in one pass, and workgroup reductions of a fixed order.
//
// With c = scale * log2(e), a row part is summed up as
//     m = max x,   s = sum 2^((x - m) c),   d = sum 2^((x - m) c) * (x - m) c         (d for the entropy alone)
// so that lse = scale m + ln s, and the entropy, ln s - ln2 d / s, adds two numbers that are not negative (d <= 0).
// Everything is fp32.  A class at -inf adds nothing; NaN and +inf make s NaN, and with it everything derived from it;
// a part in which no class is finite has m = -inf and s = 0.
#pragma once

#include "../../include/autograd_hip.h"
#include "common.hpp"

#include <math.h>

namespace agrad {

struct RowStat {
    float m, s, d;
};

__device__ __forceinline__ RowStat empty_stat() { return RowStat{-INFINITY, 0.0f, 0.0f}; }

// the same sums about the larger maximum M (M >= a.m)
template <bool ENT>
__device__ __forceinline__ RowStat about(const RowStat& a, float M, float c) {
    if (a.m == -INFINITY) return RowStat{M, a.s, a.d};           // (s is 0, or NaN and stays NaN)
    const float t = (a.m - M) * c;
    const float f = __builtin_amdgcn_exp2f(t);
    RowStat r{M, a.s * f, 0.0f};
    if constexpr (ENT) r.d = a.s == 0.0f ? 0.0f : f * __builtin_fmaf(fmaxf(t, -200.0f), a.s, a.d);
    return r;
}

template <bool ENT>
__device__ __forceinline__ RowStat merge_stat(const RowStat& a, const RowStat& b, float c) {
    const float M = fmaxf(a.m, b.m);
    const RowStat x = about<ENT>(a, M, c), y = about<ENT>(b, M, c);
    return RowStat{M, x.s + y.s, ENT ? x.d + y.d : 0.0f};
}

// A vector of a gradient to memory.  bf16: the hardware's pair conversion alone (a NaN comes out as the hardware's quiet NaN, not
// with its payload; the two compares a pair that keep it are a tenth of such a kernel's instructions).
template <typename T, int VEC>
__device__ __forceinline__ void store_grad(T* p, const float (&v)[VEC]) { VecIO<T, VEC>::store(p, v); }
template <>
__device__ __forceinline__ void store_grad<bf16_t, 8>(bf16_t* p, const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x2_hw pair = {v[2 * i], v[2 * i + 1]};
        w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, bf16x2_hw));
    }
    u32x4 t; t.x = w[0]; t.y = w[1]; t.z = w[2]; t.w = w[3];
    __builtin_nontemporal_store(t, reinterpret_cast<u32x4*>(p));
}

// one group of N values into a running part
// (returns the largest of them, -inf if none is a number)
template <bool ENT, int N>
__device__ __forceinline__ float absorb_stat(RowStat& a, const float (&v)[N], float c) {
    float top = v[0];
#pragma unroll
    for (int k = 1; k < N; ++k) top = fmaxf(top, v[k]);
    if (top > a.m) a = about<ENT>(a, top, c);
    if (a.m == -INFINITY) {                    // -inf and NaN only, so far
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (v[k] != v[k]) a.s = v[k];
        return -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const float t = (v[k] - a.m) * c;
        const float e = __builtin_amdgcn_exp2f(t);
        a.s = a.s + e;
        if constexpr (ENT) a.d = __builtin_fmaf(e, fmaxf(t, -200.0f), a.d);       // (-inf: 0 * -200)
    }
    return top;
}

// Tells the compiler that a packed vector may have changed: what it unpacked from it before is unpacked again where it is
// next needed, instead of being kept in twice the registers.
__device__ __forceinline__ void unpack_again(u32x4& r) { asm volatile("" : "+v"(r.x), "+v"(r.y), "+v"(r.z), "+v"(r.w)); }
template <typename R> __device__ __forceinline__ void unpack_again(R&) {}

// how a row of V elements that starts at `base` splits into single elements, aligned vectors, single elements
template <typename T, int VEC>
struct RowParts {
    uint32_t head, nvec, tail_start, extra;      // extra: elements outside the vectors, fewer than 2 * VEC
    __device__ __forceinline__ RowParts(const T* base, uint32_t V) {
        if constexpr (VEC == 1) {
            head = 0; nvec = V; tail_start = V; extra = 0;
        } else {
            const uint32_t mis = (uint32_t)(reinterpret_cast<uintptr_t>(base) & 15u) / (uint32_t)sizeof(T);
            head = mis ? (uint32_t)(16 / sizeof(T)) - mis : 0;
            if (head > V) head = V;
            nvec = (V - head) / VEC;
            tail_start = head + nvec * VEC;
            extra = head + (V - tail_start);
        }
    }
    // place of the i-th element outside the vectors
    __device__ __forceinline__ uint32_t extra_at(uint32_t i) const { return i < head ? i : tail_start + (i - head); }
};

// How many vectors a vector of 16 bytes stands behind a multiple of 128 bytes.  Waves that start there read and write whole lines;
// others ask for their first and last lines twice (4096 rows of 50257 fp32: 878 MB for 823, 136 against 128 us).
template <int VEC, typename T>
__device__ __forceinline__ uint32_t line_skew(const T* first) {
    return VEC == 1 ? 0u : (uint32_t)(reinterpret_cast<uintptr_t>(first) & 127u) / 16u;
}
// The same for a workgroup that takes `step` of n vectors at a time, unless one step becomes two by it.
template <int VEC, typename T>
__device__ __forceinline__ uint32_t line_skew(const T* first, uint32_t n, uint32_t step) {
    const uint32_t skew = line_skew<VEC>(first);
    return n == 0 || (n <= step && n + skew > step) ? 0u : skew;
}

// ---- a row shared by several workgroups --------------------------------------------------------------
// Where there are fewer rows than fill the GPU, `parts` workgroups take a stretch of a row's vectors each, leave what they
// found in memory that the context owns, and count themselves; the one that counts last puts the parts together.  Nobody
// waits for anybody.  The counters are zero between launches (the last one puts its counter back), and all launches of a
// context run on its one stream, recorded ones too, so that no two launches use the memory at once.
constexpr uint32_t kSharedParts = 1024;      // workgroups of a launch that share rows, at most
constexpr uint32_t kMaxParts = 32;           // parts of one row, at most
struct SharedRows {
    float* stats;             // [kSharedParts, 4]
    unsigned long long* keys; // [kSharedParts, AGRAD_MAX_TOP]
    uint32_t* tickets;        // [kSharedParts]
    float* sums;              // [kSumRows, 4], what a first pass over a row leaves for a second one of the same call
};
constexpr uint64_t kSumRows = 65536;
constexpr uint64_t kSharedRowsBytes = (uint64_t)kSharedParts * (16 + 8 * AGRAD_MAX_TOP + 4) + kSumRows * 16;

template <typename V>
__device__ __forceinline__ void put_shared(V* to, V value) { __hip_atomic_store(to, value, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename V>
__device__ __forceinline__ V get_shared(const V* from) { return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// True, in every thread, for the workgroup whose arrival is number `expected`.  What it reads with get_shared is what the
// others wrote with put_shared: device-scope stores are acknowledged once they are past the XCD's L2, every wave waits
// for the acknowledgement of its own before the barrier, and the counter moves behind the barrier.
__device__ __forceinline__ bool workgroup_arrives_last(uint32_t* ticket, uint32_t expected, uint32_t* lds_word) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");          // (keeps the compiler from moving stores down)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t old = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (old + 1u == expected) put_shared(ticket, 0u);
        *lds_word = old + 1u == expected ? 1u : 0u;
    }
    __syncthreads();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
    return *lds_word != 0u;
}

// the stretch of `part` among `parts` in n vectors
struct Stretch {
    uint32_t lo, hi;
    __device__ __forceinline__ Stretch(uint32_t n, uint32_t part, uint32_t parts) {
        const uint32_t per = (n + parts - 1) / parts;
        lo = part * per < n ? part * per : n;
        hi = lo + per < n ? lo + per : n;
    }
};

SharedRows shared_rows(void* scratch);                         // the three arrays in that memory
uint32_t row_parts(uint64_t rows, uint32_t vectors);           // how many workgroups take a row

// ---- workgroup reductions: the lanes of a wave, then the waves, in a fixed order; every thread gets the result ----
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp_move<kDppQuadXor1>(v));
    v = fmaxf(v, dpp_move<kDppQuadXor2>(v));
    v = fmaxf(v, dpp_move<kDppRowHalfMirror>(v));
    v = fmaxf(v, dpp_move<kDppRowMirror>(v));
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), kSwizzleXor16)));
    const float lo = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 0));
    const float hi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 32));
    return fmaxf(lo, hi);
}

// The maximum first, then one rescaling a thread and plain sums: a merge of two parts in each of six steps costs twelve
// exponentials.
template <int BLOCK, bool ENT>
__device__ __forceinline__ RowStat block_stat(RowStat a, float c, RowStat* lds) {
    a = about<ENT>(a, wave_max(a.m), c);
    if constexpr (ENT) wave_sum2(a.s, a.d);
    else a.s = wave_sum(a.s);
    if constexpr (BLOCK == kWave) return a;
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = a;
    __syncthreads();
    constexpr int W = BLOCK / kWave;
    if constexpr (W > 4) {                       // (sixteen waves' sums at once would be 48 registers of each thread)
        const uint32_t lane = threadIdx.x % kWave;
        a = lane < (uint32_t)W ? lds[lane] : empty_stat();
        a = about<ENT>(a, wave_max(a.m), c);
        if constexpr (ENT) wave_sum2(a.s, a.d);
        else a.s = wave_sum(a.s);
        __syncthreads();
        return a;
    }
    RowStat each[W];
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) each[w] = lds[w];
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, each[w].m);
    a = RowStat{M, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const RowStat x = about<ENT>(each[w], M, c);
        a.s = a.s + x.s;
        if constexpr (ENT) a.d = a.d + x.d;
    }
    __syncthreads();
    return a;
}

template <int BLOCK>
__device__ __forceinline__ float block_total(float v, float* lds) {
    v = wave_sum(v);
    if constexpr (BLOCK > kWave) {
        if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int w = 1; w < BLOCK / kWave; ++w) v = v + lds[w];
        __syncthreads();
    }
    return v;
}

template <int BLOCK>
__device__ __forceinline__ float block_largest(float v, float* lds) {
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) v = fmaxf(v, __shfl_xor(v, off));
    if constexpr (BLOCK > kWave) {
        if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int w = 1; w < BLOCK / kWave; ++w) v = fmaxf(v, lds[w]);
        __syncthreads();
    }
    return v;
}

}  // namespace agrad
