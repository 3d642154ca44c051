// Device parts shared by the operators that read rows of logits (logprobs.hip, distill.hip): the statistics of a
// softmax over scale * x in one pass, and workgroup reductions of a fixed order.
//
// With c = scale * log2(e), a row part is summed up as
//     m = max x,   s = sum 2^((x - m) c),   d = sum 2^((x - m) c) * (x - m) c         (d for the entropy alone)
// so that lse = scale m + ln s, and the entropy, ln s - ln2 d / s, adds two numbers that are not negative (d <= 0).
// Everything is fp32.  A class at -inf adds nothing; NaN and +inf make s NaN, and with it everything derived from it;
// a part in which no class is finite has m = -inf and s = 0.
#pragma once

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

// one group of N values into a running part
template <bool ENT, int N>
__device__ __forceinline__ void absorb_stat(RowStat& a, const float (&v)[N], float c) {
    float top = v[0];
#pragma unroll
    for (int k = 1; k < N; ++k) top = fmaxf(top, v[k]);
    if (top > a.m) a = about<ENT>(a, top, c);
    if (a.m == -INFINITY) {                    // -inf and NaN only, so far
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (v[k] != v[k]) a.s = v[k];
        return;
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const float t = (v[k] - a.m) * c;
        const float e = __builtin_amdgcn_exp2f(t);
        a.s = a.s + e;
        if constexpr (ENT) a.d = __builtin_fmaf(e, fmaxf(t, -200.0f), a.d);       // (-inf: 0 * -200)
    }
}

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

// ---- workgroup reductions: lanes by butterflies, then the waves in order; every thread gets the result ----
template <int BLOCK, bool ENT>
__device__ __forceinline__ RowStat block_stat(RowStat a, float c, RowStat* lds) {
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        RowStat o{__shfl_xor(a.m, off), __shfl_xor(a.s, off), ENT ? __shfl_xor(a.d, off) : 0.0f};
        a = merge_stat<ENT>(a, o, c);
    }
    if constexpr (BLOCK == kWave) return a;
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = a;
    __syncthreads();
    a = lds[0];
#pragma unroll
    for (int w = 1; w < BLOCK / kWave; ++w) a = merge_stat<ENT>(a, lds[w], c);
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
