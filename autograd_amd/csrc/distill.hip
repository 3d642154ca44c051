// Distillation from a teacher's top logits: the Kullback-Leibler divergence of the student's distribution
// p = softmax(scale * x) from a teacher's q, of which `top` classes a row are known, and its gradient.
//
//   RENORM   q = softmax(teacher_scale * u) over the row's used slots
//            loss = sum_k q_k (log q_k - log p[id_k])
//   TAIL     q_k = exp(u_k), the values are log probabilities; what they leave, q_rest = max(0, 1 - sum q), belongs to
//            all the other classes together, to which the student gives p_rest = sum of p outside the ids
//            loss = sum_k q_k (log q_k - log p[id_k]) + q_rest (log q_rest - log p_rest)
//   gradient with W = sum q + q_rest, r = softmax of z over the classes outside the ids:
//            d loss / d z[v] = p[v] W - sum of the q_k with id_k == v     among the ids
//                              p[v] W                                     elsewhere, RENORM
//                              r[v] (W p_rest - q_rest)                   elsewhere, TAIL
//            dx = scale * (d loss / d z) * upstream
//
// The classes outside the ids are summed up on their own, not as 1 - sum p[id]: a student that is sure of itself has a
// p_rest far below the rounding of 1, down to below the smallest number.  The test for "outside" costs a row's stream one
// look at an LDS bit a vector.
#include "launch.hpp"
#include "row_softmax.hpp"

#include <cmath>

namespace agrad {

namespace {

constexpr int kDsBlock = 256;
constexpr int kDsUnroll = 4;
constexpr uint32_t kSetWords = 512;          // bits of the vectors that hold an id, by the vector's number modulo 16384
static_assert(AGRAD_MAX_TOP <= kDsBlock, "a thread a teacher slot");

struct DsArgs {
    const int32_t* ids; const float* values;
    uint64_t ld; uint32_t V, top; float scale, c, teacher_scale; uint32_t tail;
    int* err_flag;
};
struct DsOut {
    float* loss; float* stats;                                     // forward
    const float* row_scale; float grad_scale;                      // loss and gradient in one launch
};

// a row's teacher slots in LDS: the class of each (-1: unused), its probability, log probability
struct Slots {
    int32_t id[AGRAD_MAX_TOP];
    float q[AGRAD_MAX_TOP];
    uint32_t bits[kSetWords];
};

__device__ __forceinline__ bool set_bit(const Slots& s, uint32_t vec) {
    return (s.bits[(vec >> 5) & (kSetWords - 1)] >> (vec & 31u)) & 1u;
}

__device__ __forceinline__ int32_t slot_id(const DsArgs& a, uint64_t row, uint32_t k, bool report) {
    if (k >= a.top) return -1;
    const int32_t id = a.ids[row * a.top + k];
    if (id >= 0 && (uint32_t)id < a.V) return id;
    if (report && id != -1) *a.err_flag = 1;
    return -1;
}

// The teacher's side of a row, thread k its slot k: log q (of an unused slot -inf), and for everyone sum q (0: no slots)
// and, in RENORM, the log of the softmax's denominator.
struct Teacher {
    float log_q, mass, lse;
};
template <int BLOCK>
__device__ __forceinline__ Teacher teacher_row(const DsArgs& a, uint64_t row, int32_t id, float* lds) {
    const float u = id >= 0 ? a.values[row * a.top + threadIdx.x] : -INFINITY;
    Teacher t;
    if (a.tail) {
        t.log_q = u;
        t.lse = 0.0f;
        t.mass = block_total<BLOCK>(expf(u), lds);
        return t;
    }
    const float w = id >= 0 ? u * a.teacher_scale : -INFINITY;
    const float m = block_largest<BLOCK>(w, lds);
    const float e = m == -INFINITY ? (w != w ? w : 0.0f) : expf(w - m);
    const float total = block_total<BLOCK>(e, lds);
    if (total == 0.0f) return Teacher{-INFINITY, 0.0f, INFINITY};         // no slots: nothing to learn from
    t.lse = m + logf(total);
    t.log_q = w - t.lse;
    t.mass = 1.0f;
    return t;
}

// marks the vectors that hold an id
template <int VEC>
__device__ __forceinline__ void mark_slots(Slots& s, int32_t id, uint32_t head, uint32_t nvec) {
    if (id >= (int32_t)head) {
        const uint32_t vec = ((uint32_t)id - head) / VEC;
        if (vec < nvec) atomicOr(&s.bits[(vec >> 5) & (kSetWords - 1)], 1u << (vec & 31u));
    }
}

// The student's side of a row: all classes, and in TAIL those outside the ids.
struct Student {
    RowStat all, rest;
};
template <typename T, int VEC, int BLOCK, bool TAIL>
__device__ __forceinline__ Student student_row(const T* base, const DsArgs& a, const Slots& slots, int32_t id, float at, bool first,
                                               RowStat* lds) {
    const RowParts<T, VEC> parts(base, a.V);
    RowStat r = empty_stat();
    if (threadIdx.x < parts.extra) {
        const uint32_t e = parts.extra_at(threadIdx.x);
        float v[1];
        VecIO<T, 1>::load(base + e, v);
        if (TAIL)
            for (uint32_t k = 0; k < a.top; ++k)
                if (slots.id[k] == (int32_t)e) v[0] = -INFINITY;
        absorb_stat<false, 1>(r, v, a.c);
    }
    const T* body = base + parts.head;
    for (uint32_t i0 = threadIdx.x; i0 < parts.nvec; i0 += BLOCK * kDsUnroll) {
        float v[kDsUnroll][VEC];
#pragma unroll
        for (int u = 0; u < kDsUnroll; ++u) {
            const uint32_t i = i0 + u * BLOCK;
            if (i < parts.nvec) VecIO<T, VEC>::load(body + (uint64_t)i * VEC, v[u]);
        }
#pragma unroll
        for (int u = 0; u < kDsUnroll; ++u) {
            const uint32_t i = i0 + u * BLOCK;
            if (i >= parts.nvec) continue;
            if (TAIL && set_bit(slots, i)) {
                const uint32_t e = parts.head + i * VEC;
                for (uint32_t k = 0; k < a.top; ++k) {
                    const uint32_t off = (uint32_t)slots.id[k] - e;
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        if (off == (uint32_t)j) v[u][j] = -INFINITY;
                }
            }
            absorb_stat<false, VEC>(r, v[u], a.c);
        }
    }
    r = block_stat<BLOCK, false>(r, a.c, lds);
    if (!TAIL) return Student{r, r};
    // the ids' own classes, each once
    RowStat own = empty_stat();
    if (id >= 0 && first) {
        float v[1] = {at};
        absorb_stat<false, 1>(own, v, a.c);
    }
    own = block_stat<BLOCK, false>(own, a.c, lds);
    return Student{merge_stat<false>(r, own, a.c), r};
}

// What a row's gradient is made of: the classes outside the ids have exp(z - lse_out) out, those among them
// exp(z - lse) mass - q.  lse = -inf: the row has no gradient.
struct RowGrad {
    float lse, lse_out, mass, out;
};

// Everything of a row but its gradient: the slots in LDS, the loss, and what the gradient needs.
template <typename T, int VEC, int BLOCK, bool TAIL>
__device__ __forceinline__ RowGrad row_loss(const T* base, uint64_t row, const DsArgs& a, Slots& slots, float* lds, RowStat* lds_stat,
                                            float* loss_out, float& teacher_lse) {
    const RowParts<T, VEC> parts(base, a.V);
    const uint32_t k = threadIdx.x;
    const int32_t id = slot_id(a, row, k, true);
    float at[1];                                   // the student's logit of this thread's slot
    VecIO<T, 1>::load(base + (id >= 0 ? id : 0), at);
    for (uint32_t i = k; i < kSetWords; i += BLOCK) slots.bits[i] = 0;
    const bool used = __syncthreads_or(id >= 0) != 0;
    const Teacher t = teacher_row<BLOCK>(a, row, id, lds);
    const float q = expf(t.log_q);
    if (k < AGRAD_MAX_TOP) {
        slots.id[k] = id;
        slots.q[k] = q;
    }
    __syncthreads();
    mark_slots<VEC>(slots, id, parts.head, parts.nvec);
    bool first = true;
    if (TAIL && id >= 0)
        for (uint32_t j = 0; j < k; ++j) first = first && slots.id[j] != id;
    __syncthreads();
    const Student s = student_row<T, VEC, BLOCK, TAIL>(base, a, slots, id, at[0], first, lds_stat);
    const bool none = !used || t.lse == INFINITY || (s.all.m == -INFINITY && s.all.s == 0.0f);
    const float log_s = logf(s.all.s);
    float term = 0.0f;
    if (id >= 0 && !(q == 0.0f)) term = q * (t.log_q - ((at[0] - s.all.m) * a.scale - log_s));
    float loss = block_total<BLOCK>(term, lds);
    RowGrad g;
    g.lse = s.all.m * a.scale + log_s;
    g.lse_out = g.lse;
    g.mass = t.mass;
    g.out = t.mass;
    if (TAIL) {
        if (s.rest.m == -INFINITY && s.rest.s == 0.0f) {       // no class outside the ids has mass
            g.lse_out = INFINITY;
        } else {
            const float q_rest = fmaxf(1.0f - t.mass, 0.0f), log_rest = logf(s.rest.s);
            const float log_p_rest = (s.rest.m - s.all.m) * a.scale + (log_rest - log_s);
            if (q_rest > 0.0f) loss = loss + q_rest * (logf(q_rest) - log_p_rest);
            g.lse_out = s.rest.m * a.scale + log_rest;
            g.mass = t.mass + q_rest;
            g.out = g.mass * expf(log_p_rest) - q_rest;
        }
    }
    teacher_lse = t.lse;
    if (none) {
        loss = 0.0f;
        g = RowGrad{-INFINITY, INFINITY, 0.0f, 0.0f};
    }
    if (k == 0 && loss_out != nullptr) loss_out[row] = loss;
    return g;
}

// one vector of the gradient: first: its first class; near: it may hold an id
template <int VEC>
__device__ __forceinline__ void ds_grad(float (&v)[VEC], const RowGrad& g, float scale, float mul, uint32_t first, bool near, const int32_t* id,
                                        const float* q, uint32_t n) {
    float x[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        x[j] = v[j] * scale;
        v[j] = __builtin_amdgcn_exp2f((x[j] - g.lse_out) * kLog2eHi) * g.out;
    }
    if (near) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            bool in_set = false;
            float taken = 0.0f;
            for (uint32_t k = 0; k < n; ++k) {
                if ((uint32_t)id[k] == first + (uint32_t)j) {
                    in_set = true;
                    taken = taken + q[k];
                }
            }
            if (in_set) v[j] = __builtin_amdgcn_exp2f((x[j] - g.lse) * kLog2eHi) * g.mass - taken;
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = v[j] * mul;
}

// (a row without a gradient: zeros, whatever its logits hold)
template <int VEC>
__device__ __forceinline__ void ds_zero(float (&v)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = 0.0f;
}

template <typename T, int VEC>
__device__ __forceinline__ void ds_store(T* to, float (&d)[VEC], uint32_t accumulate) {
    if (accumulate) {
        float old[VEC];
        VecIO<T, VEC>::load(to, old);
#pragma unroll
        for (int k = 0; k < VEC; ++k) d[k] = old[k] + d[k];
    }
    VecIO<T, VEC>::store(to, d);
}

template <typename T, int VEC, bool TAIL>
__global__ void __launch_bounds__(kDsBlock)
distill_fwd_kernel(const T* __restrict__ x, const DsArgs a, const DsOut o) {
    __shared__ Slots slots;
    __shared__ float lds[kDsBlock / kWave];
    __shared__ RowStat lds_stat[kDsBlock / kWave];
    const uint64_t row = blockIdx.x;
    float teacher_lse;
    const RowGrad g = row_loss<T, VEC, kDsBlock, TAIL>(x + row * a.ld, row, a, slots, lds, lds_stat, o.loss, teacher_lse);
    if (threadIdx.x == 0 && o.stats != nullptr) {
        float* to = o.stats + row * 4;
        to[0] = g.lse; to[1] = TAIL ? g.lse_out : teacher_lse; to[2] = g.mass; to[3] = g.out;
    }
}

// loss and gradient of a row in one workgroup (x and dx may be the same memory)
template <typename T, int VEC, bool TAIL>
__global__ void __launch_bounds__(kDsBlock)
distill_fused_kernel(const T* x, T* dx, const DsArgs a, const DsOut o) {
    __shared__ Slots slots;
    __shared__ float lds[kDsBlock / kWave];
    __shared__ RowStat lds_stat[kDsBlock / kWave];
    const uint64_t row = blockIdx.x;
    const T* base = x + row * a.ld;
    T* out = dx + row * a.ld;
    float teacher_lse;
    const RowGrad g = row_loss<T, VEC, kDsBlock, TAIL>(base, row, a, slots, lds, lds_stat, o.loss, teacher_lse);
    const float mul = a.scale * (o.row_scale != nullptr ? o.row_scale[row] : o.grad_scale);
    const bool none = g.lse == -INFINITY;
    const RowParts<T, VEC> parts(base, a.V);
    if (threadIdx.x < parts.extra) {
        const uint32_t e = parts.extra_at(threadIdx.x);
        float v[1];
        VecIO<T, 1>::load(base + e, v);
        if (none) ds_zero<1>(v);
        else ds_grad<1>(v, g, a.scale, mul, e, true, slots.id, slots.q, a.top);
        VecIO<T, 1>::store(out + e, v);
    }
    for (uint32_t i = threadIdx.x; i < parts.nvec; i += kDsBlock) {
        const uint32_t e = parts.head + i * VEC;
        float v[VEC];
        VecIO<T, VEC>::load(base + e, v);
        if (none) ds_zero<VEC>(v);
        else ds_grad<VEC>(v, g, a.scale, mul, e, set_bit(slots, i), slots.id, slots.q, a.top);
        VecIO<T, VEC>::store(out + e, v);
    }
}

// the gradient with the row's statistics given: a workgroup a chunk of a row
template <typename T, int VEC>
__global__ void __launch_bounds__(kDsBlock)
distill_bwd_kernel(const T* x, T* dx, const DsArgs a, const float* dloss, const float* stats, uint32_t accumulate, const FastDiv32 chunks) {
    __shared__ int32_t ids[AGRAD_MAX_TOP];
    __shared__ float qs[AGRAD_MAX_TOP];
    __shared__ uint32_t in_wave[2];
    const uint32_t row = chunks.div(blockIdx.x), chunk = blockIdx.x - row * chunks.d, tid = threadIdx.x;
    const T* base = x + (uint64_t)row * a.ld;
    T* out = dx + (uint64_t)row * a.ld;
    const RowParts<T, VEC> parts(base, a.V);
    const uint32_t span = kDsBlock * kDsUnroll;                      // vectors of a chunk
    float v[kDsUnroll][VEC];
#pragma unroll
    for (int u = 0; u < kDsUnroll; ++u) {
        const uint32_t i = chunk * span + u * kDsBlock + tid;
        if (i < parts.nvec) VecIO<T, VEC>::load(base + parts.head + (uint64_t)i * VEC, v[u]);
    }
    const float* st = stats + (uint64_t)row * 4;
    const RowGrad g{st[0], a.tail ? st[1] : st[0], st[2], st[3]};
    const float teacher_lse = st[1];
    const float mul = a.scale * dloss[row];
    const bool none = g.lse == -INFINITY;
    // the slots whose class lies in this chunk (chunk 0: or outside the vectors), in slot order
    static_assert(AGRAD_MAX_TOP <= 2 * kWave, "the slots of two waves");
    const int32_t id = slot_id(a, row, tid, chunk == 0);
    const uint32_t vec = id >= (int32_t)parts.head ? ((uint32_t)id - parts.head) / VEC : 0xffffffffu;
    const bool outside_vectors = id >= 0 && vec >= parts.nvec;
    const bool here = !none && id >= 0 && (outside_vectors ? chunk == 0 : vec / span == chunk);
    const uint64_t lanes = __ballot(here);
    if (tid < 2 * kWave && tid % kWave == 0) in_wave[tid / kWave] = (uint32_t)__popcll(lanes);
    __syncthreads();
    if (here) {
        const uint32_t at = (tid >= kWave ? in_wave[0] : 0u) + (uint32_t)__popcll(lanes & ((1ull << (tid % kWave)) - 1));
        const float u = a.values[(uint64_t)row * a.top + tid];
        ids[at] = id;
        qs[at] = a.tail ? expf(u) : expf(u * a.teacher_scale - teacher_lse);
    }
    __syncthreads();
    const uint32_t n = in_wave[0] + in_wave[1];
    if (chunk == 0 && tid < parts.extra) {
        const uint32_t e = parts.extra_at(tid);
        float w[1];
        VecIO<T, 1>::load(base + e, w);
        if (none) ds_zero<1>(w);
        else ds_grad<1>(w, g, a.scale, mul, e, true, ids, qs, n);
        ds_store<T, 1>(out + e, w, accumulate);
    }
#pragma unroll
    for (int u = 0; u < kDsUnroll; ++u) {
        const uint32_t i = chunk * span + u * kDsBlock + tid;
        if (i >= parts.nvec) continue;
        const uint32_t e = parts.head + i * VEC;
        bool near = false;
        for (uint32_t k = 0; k < n; ++k) near = near || (uint32_t)ids[k] - e < (uint32_t)VEC;
        if (none) ds_zero<VEC>(v[u]);
        else ds_grad<VEC>(v[u], g, a.scale, mul, e, near, ids, qs, n);
        ds_store<T, VEC>(out + e, v[u], accumulate);
    }
}

template <typename T>
int ds_fwd_typed(hipStream_t s, const T* x, const DsArgs& a, const DsOut& o, uint64_t rows) {
    constexpr int WIDE = WideVec<T>::value;
    const bool wide = a.V >= 4 * WIDE;
    const dim3 grid((uint32_t)rows), block(kDsBlock);
    if (wide && a.tail) hipLaunchKernelGGL((distill_fwd_kernel<T, WIDE, true>), grid, block, 0, s, x, a, o);
    else if (wide) hipLaunchKernelGGL((distill_fwd_kernel<T, WIDE, false>), grid, block, 0, s, x, a, o);
    else if (a.tail) hipLaunchKernelGGL((distill_fwd_kernel<T, 1, true>), grid, block, 0, s, x, a, o);
    else hipLaunchKernelGGL((distill_fwd_kernel<T, 1, false>), grid, block, 0, s, x, a, o);
    return check_hip(hipGetLastError(), "top-k distillation launch");
}

inline bool one_alignment(const void* x, const void* dx) {
    return ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15u) == 0;
}

template <typename T>
int ds_fused_typed(hipStream_t s, const T* x, T* dx, const DsArgs& a, const DsOut& o, uint64_t rows) {
    constexpr int WIDE = WideVec<T>::value;
    const bool wide = a.V >= 4 * WIDE && one_alignment(x, dx);
    const dim3 grid((uint32_t)rows), block(kDsBlock);
    if (wide && a.tail) hipLaunchKernelGGL((distill_fused_kernel<T, WIDE, true>), grid, block, 0, s, x, dx, a, o);
    else if (wide) hipLaunchKernelGGL((distill_fused_kernel<T, WIDE, false>), grid, block, 0, s, x, dx, a, o);
    else if (a.tail) hipLaunchKernelGGL((distill_fused_kernel<T, 1, true>), grid, block, 0, s, x, dx, a, o);
    else hipLaunchKernelGGL((distill_fused_kernel<T, 1, false>), grid, block, 0, s, x, dx, a, o);
    return check_hip(hipGetLastError(), "top-k distillation launch");
}

template <typename T>
int ds_bwd_typed(hipStream_t s, const T* x, T* dx, const DsArgs& a, const float* dloss, const float* stats, uint32_t accumulate,
                 uint64_t rows) {
    constexpr int WIDE = WideVec<T>::value;
    const bool wide = a.V >= 4 * WIDE && one_alignment(x, dx);
    const uint32_t vec = wide ? WIDE : 1, span = kDsBlock * kDsUnroll;
    const uint32_t chunks = (a.V / vec + span - 1) / span;
    uint64_t max_rows = 0x00ffffffull / chunks;                  // workgroups of a launch: 2^32 threads
    if (max_rows == 0) max_rows = 1;
    for (uint64_t r0 = 0; r0 < rows; r0 += max_rows) {
        const uint64_t n = rows - r0 < max_rows ? rows - r0 : max_rows;
        DsArgs b = a;
        b.ids += r0 * a.top;
        b.values += r0 * a.top;
        const dim3 grid((uint32_t)(n * chunks)), block(kDsBlock);
        if (wide) hipLaunchKernelGGL((distill_bwd_kernel<T, WIDE>), grid, block, 0, s, x + r0 * a.ld, dx + r0 * a.ld, b, dloss + r0, stats + 4 * r0, accumulate, FastDiv32(chunks));
        else hipLaunchKernelGGL((distill_bwd_kernel<T, 1>), grid, block, 0, s, x + r0 * a.ld, dx + r0 * a.ld, b, dloss + r0, stats + 4 * r0, accumulate, FastDiv32(chunks));
    }
    return check_hip(hipGetLastError(), "top-k distillation backward launch");
}

int ds_args(const char* what, int dtype, const void* logits, const int32_t* ids, const float* values, const void* dlogits,
            uint64_t rows, uint32_t V, uint64_t ld, uint32_t top, float scale, float teacher_scale, int mode, int* err_flag, DsArgs* a) {
    if (int rc = logits_check(what, dtype, logits, dlogits, rows, V, ld, scale)) return rc;
    if (mode != AGRAD_DISTILL_RENORM && mode != AGRAD_DISTILL_TAIL) return set_error(AGRAD_EINVAL, "%s: unknown mode %d", what, mode);
    if (top == 0 || top > AGRAD_MAX_TOP) return set_error(AGRAD_EINVAL, "%s: 1 to %u teacher slots a row, got %u", what, AGRAD_MAX_TOP, top);
    if (!(teacher_scale > 0.0f) || !std::isfinite(teacher_scale))
        return set_error(AGRAD_EINVAL, "%s: the teacher's scale must be positive and finite", what);
    if (mode == AGRAD_DISTILL_TAIL && teacher_scale != 1.0f)
        return set_error(AGRAD_EINVAL, "%s: log probabilities with a tail are taken as they are (teacher_scale 1)", what);
    if (rows != 0 && (logits == nullptr || ids == nullptr || values == nullptr)) return set_error(AGRAD_EINVAL, "%s: null operand", what);
    const float c = (float)((double)scale * 1.4426950408889634);
    *a = DsArgs{ids, values, ld, V, top, scale, c, teacher_scale, mode == AGRAD_DISTILL_TAIL ? 1u : 0u, err_flag};
    return AGRAD_OK;
}

}  // namespace

int launch_distill_fwd(hipStream_t s, int dtype, const void* logits, const int32_t* ids, const float* values, float* loss, float* stats,
                       uint64_t rows, uint32_t V, uint64_t ld, uint32_t top, float scale, float teacher_scale, int mode, int* err_flag) {
    DsArgs a;
    if (int rc = ds_args("top-k distillation", dtype, logits, ids, values, nullptr, rows, V, ld, top, scale, teacher_scale, mode, err_flag, &a)) return rc;
    if (rows == 0) return AGRAD_OK;
    if (loss == nullptr) return set_error(AGRAD_EINVAL, "top-k distillation: null loss");
    const DsOut o{loss, stats, nullptr, 0.0f};
    if (dtype == AGRAD_F32) return ds_fwd_typed<float>(s, (const float*)logits, a, o, rows);
    return ds_fwd_typed<bf16_t>(s, (const bf16_t*)logits, a, o, rows);
}

int launch_distill_bwd(hipStream_t s, int dtype, const void* logits, const int32_t* ids, const float* values, const float* dloss,
                       const float* stats, void* dlogits, uint64_t rows, uint32_t V, uint64_t ld, uint32_t top, float scale,
                       float teacher_scale, int mode, uint32_t flags, int* err_flag) {
    DsArgs a;
    if (int rc = ds_args("top-k distillation backward", dtype, logits, ids, values, dlogits, rows, V, ld, top, scale, teacher_scale, mode, err_flag, &a)) return rc;
    if (flags & ~(uint32_t)AGRAD_ACC_INPUT_GRAD) return set_error(AGRAD_EINVAL, "top-k distillation backward: unknown flag bits 0x%x", flags);
    if (rows == 0) return AGRAD_OK;
    if (dloss == nullptr || stats == nullptr || dlogits == nullptr) return set_error(AGRAD_EINVAL, "top-k distillation backward: null operand");
    const uint32_t acc = (flags & AGRAD_ACC_INPUT_GRAD) ? 1u : 0u;
    if (dtype == AGRAD_F32) return ds_bwd_typed<float>(s, (const float*)logits, (float*)dlogits, a, dloss, stats, acc, rows);
    return ds_bwd_typed<bf16_t>(s, (const bf16_t*)logits, (bf16_t*)dlogits, a, dloss, stats, acc, rows);
}

int launch_distill_fused(hipStream_t s, int dtype, const void* logits, const int32_t* ids, const float* values, float* loss,
                         const float* row_scale, void* dlogits, uint64_t rows, uint32_t V, uint64_t ld, uint32_t top, float scale,
                         float teacher_scale, float grad_scale, int mode, int* err_flag) {
    DsArgs a;
    if (int rc = ds_args("top-k distillation step", dtype, logits, ids, values, dlogits, rows, V, ld, top, scale, teacher_scale, mode, err_flag, &a)) return rc;
    if (rows == 0) return AGRAD_OK;
    if (dlogits == nullptr) return set_error(AGRAD_EINVAL, "top-k distillation step: null gradient");
    const DsOut o{loss, nullptr, row_scale, grad_scale};
    if (dtype == AGRAD_F32) return ds_fused_typed<float>(s, (const float*)logits, (float*)dlogits, a, o, rows);
    return ds_fused_typed<bf16_t>(s, (const bf16_t*)logits, (bf16_t*)dlogits, a, o, rows);
}

}  // namespace agrad
