// Distillation from a teacher's top logits: the Kullback-Leibler divergence of the student's distribution
// p = softmax(scale * x) from a teacher's q, of which `top` classes a row are known, and its gradient.
//
//   RENORM   q = softmax(teacher_scale * u) over the row's used slots, about the largest u
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
// p_rest far below the rounding of 1, down to below the smallest number.  For that the ids of a row are marked in a bit map
// in LDS, a bit a class, and a vector of logits looks its bits up: three instructions a vector of 16 bytes.  The gradient
// treats all classes as classes outside, and the few among the ids are stored over that.
//
// HBM bounds all of it: the forward pass reads the logits once, the backward pass reads them and writes the gradient, and
// loss and gradient in one launch read once and write once where a workgroup's registers hold the row.
#include "launch.hpp"
#include "row_softmax.hpp"

#include <cmath>

namespace agrad {

namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
constexpr int kDsBlock = 256;
constexpr int kDsUnroll = 4;                       // vectors a thread keeps in flight
constexpr uint32_t kMapWords = 5120;               // of the bit map: 163840 classes of a row, or of a part of one
constexpr uint32_t kMapBits = kMapWords * 32;
constexpr uint32_t kShortMap = 2048;               // words: 65536 classes
static_assert(AGRAD_MAX_TAIL_CLASSES == kMaxParts * kMapBits, "a row's parts hold the bits of so many classes");
static_assert(AGRAD_MAX_TOP <= kDsBlock && AGRAD_MAX_TOP == 2 * kWave, "a thread a teacher slot, the slots of two waves");

struct DsArgs {
    const int32_t* ids; const float* values;
    uint64_t ld; uint32_t V, top; float scale, c, teacher_scale;
    int* err_flag;
};
struct DsOut {
    float* loss; float* stats;                     // forward
    const float* row_scale; float grad_scale;      // loss and gradient in one launch
    SharedRows shared; uint32_t parts;
};

// ---- the bit map of a row's ids -----------------------------------------------------------------------
template <int BLOCK>
__device__ __forceinline__ void clear_map(uint32_t* map, uint32_t classes) {
    const uint32_t n = (classes + 127) / 128;
    for (uint32_t i = threadIdx.x; i < n; i += BLOCK) reinterpret_cast<u32x4*>(map)[i] = u32x4{0u, 0u, 0u, 0u};
}
// (the bits of a stretch of the row's vectors, and a word for the elements outside the vectors)
template <typename P>
__device__ __forceinline__ void mark(uint32_t* map, uint32_t& outside, const P& parts, int32_t id, uint32_t first, uint32_t classes) {
    if (id < 0) return;
    const uint32_t at = (uint32_t)id - first;
    if ((uint32_t)id < parts.head) atomicOr(&outside, 1u << id);
    else if (at < classes) atomicOr(&map[at / 32], 1u << (at % 32));
    else if ((uint32_t)id >= parts.tail_start) atomicOr(&outside, 1u << (parts.head + ((uint32_t)id - parts.tail_start)));
}
// the bits of the vec-th vector
template <int VEC>
__device__ __forceinline__ uint32_t bits_of(const uint32_t* map, uint32_t vec) {
    const uint32_t at = vec * VEC;
    return (map[at / 32] >> (at % 32)) & ((1u << VEC) - 1u);
}
__device__ __forceinline__ void mask_raw(f32x4& r, uint32_t bits) {
    if (bits & 1u) r.x = -INFINITY;
    if (bits & 2u) r.y = -INFINITY;
    if (bits & 4u) r.z = -INFINITY;
    if (bits & 8u) r.w = -INFINITY;
}
__device__ __forceinline__ uint32_t mask_pair(uint32_t w, uint32_t bits) {
    if (bits & 1u) w = (w & 0xffff0000u) | 0xff80u;
    if (bits & 2u) w = (w & 0x0000ffffu) | 0xff800000u;
    return w;
}
__device__ __forceinline__ void mask_raw(u32x4& r, uint32_t bits) {
    r.x = mask_pair(r.x, bits);
    r.y = mask_pair(r.y, bits >> 2);
    r.z = mask_pair(r.z, bits >> 4);
    r.w = mask_pair(r.w, bits >> 6);
}
__device__ __forceinline__ void mask_raw(float& r, uint32_t bits) { if (bits) r = -INFINITY; }
__device__ __forceinline__ void mask_raw(bf16_t& r, uint32_t bits) { if (bits) r = 0xff80; }

// ---- the teacher's side of a row ------------------------------------------------------------------------
// Thread k has slot k, with the value u (-inf, if unused): log q.  For everyone: sum q, and of the softmax (RENORM) its largest
// value and the log of its sum about that (+inf: no slots to learn from).  The two are kept apart: together they would be rounded at the
// size of the values, whose common offset is no part of q (64 values of 1e6: log q off by 0.03).
struct Teacher {
    float log_q, mass, top, log_sum;
};
// log q of a value: distances to the largest first
__device__ __forceinline__ float renorm_log_q(float u, float top, float log_sum, float teacher_scale) { return (u - top) * teacher_scale - log_sum; }
template <int BLOCK, bool TAIL>
__device__ __forceinline__ Teacher teacher_row(const DsArgs& a, float u, float* lds) {
    if (TAIL) return Teacher{u, block_total<BLOCK>(expf(u), lds), 0.0f, 0.0f};
    const float top = block_largest<BLOCK>(u, lds);
    const float e = top == -INFINITY ? (u != u ? u : 0.0f) : expf((u - top) * a.teacher_scale);
    const float total = block_total<BLOCK>(e, lds);
    if (total == 0.0f) return Teacher{-INFINITY, 0.0f, -INFINITY, INFINITY};
    const float log_sum = logf(total);
    // (sum q is 1; NaN for a value of NaN or +inf)
    return Teacher{renorm_log_q(u, top, log_sum, a.teacher_scale), total == total ? 1.0f : total, top, log_sum};
}

// Slots in LDS.  A class that a row names twice counts with both its q; only its first slot stands for it.
struct Slots {
    __align__(16) int32_t id[AGRAD_MAX_TOP];         // (unused slots, and those past the row's: -1)
    __align__(16) float q[AGRAD_MAX_TOP];
};
struct Own {
    bool first;
    float taken;              // sum of the q of this slot's class, in slot order
};
// (every slot against all: eight at a time and without a branch, so that the reads follow one another without a wait.  One slot at
// a time, leaving early, took 4 us of a row's latency with 64 ids; sixteen at a time take a workgroup of 1024 threads more than
// 64 registers, and a CU its second one.)
template <bool TAKEN>
__device__ __forceinline__ Own own_slot(const Slots& s, uint32_t n, uint32_t k, int32_t id) {
    uint32_t at = 0xffffffffu;
    float taken = 0.0f;
    if (__ballot(id >= 0) != 0)
#pragma unroll 2
        for (uint32_t j = 0; j < n; j += 4) {
            const i32x4 ids = *reinterpret_cast<const i32x4*>(s.id + j);
            f32x4 q = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (TAKEN) q = *reinterpret_cast<const f32x4*>(s.q + j);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool same = ids[i] == id;
                if constexpr (TAKEN) taken = taken + (same ? q[i] : 0.0f);
                at = same && j + i < at ? j + i : at;
            }
        }
    return Own{id >= 0 && at == k, taken};
}

// Who stores a class: a list of slots for each thread of a group, which stores them after its vectors.  The slots of one class are
// in one thread's list; the order of a list, which atomics decide, does not matter.
template <int THREADS>
struct PatchLists {
    uint32_t head[THREADS];
    uint32_t next[AGRAD_MAX_TOP];
    int32_t id[AGRAD_MAX_TOP];
    float value[AGRAD_MAX_TOP];
    static constexpr uint32_t kNone = 0xffffffffu;
    __device__ __forceinline__ void add(uint32_t slot, uint32_t thread, int32_t cls, float v) {
        id[slot] = cls;
        value[slot] = v;
        next[slot] = atomicExch(&head[thread], slot);
    }
    template <typename T>
    __device__ __forceinline__ void store(T* out, uint32_t thread) const {
        for (uint32_t j = head[thread]; j != kNone; j = next[j]) {
            float d[1] = {value[j]};
            VecIO<T, 1>::store(out + id[j], d);
        }
    }
};

// ---- what a row's gradient is made of --------------------------------------------------------------------
// Where p_rest is below fp32's numbers, down to classes at a mask's lowest value, the sums about m say nothing of the classes outside.
// There a forward call leaves, in place of log p_rest and sum q, their own largest logit and -1 - the log of their sum about it; sum q
// is negative in no other row.
constexpr float kFarRest = -100.0f;                    // log p_rest, with fp32's error of 2^-17 in it
// all: log of the student's whole sum about m, the largest logit (m = -inf: no gradient); log_rest: log of p_rest (TAIL;
// -inf: no class outside), mass: sum q.  This is what a forward call leaves for its backward call, so that a row of logits
// far from 0 loses nothing (an lse of 1e6 would have lost log p).  A row whose loss is NaN has NaN in all four, so that its whole
// gradient is NaN: its largest logit alone may be -inf, which would say that there is none.
struct RowSums {
    float m, all, log_rest, mass;
};
struct RowGrad {
    float m;
    float out_log, out;       // outside the ids:  out exp((x - m) scale - out_log)
    float all, mass;          // among them:       mass exp((x - m) scale - all) - q
};
template <bool TAIL>
__device__ __forceinline__ RowGrad row_grad(const RowSums& s) {
    RowGrad g{s.m, s.all, s.mass, s.all, s.mass};
    if (TAIL) {
        if (s.log_rest == -INFINITY) {
            g.out = 0.0f;                                          // no class outside has mass
        } else {
            const float q_rest = fmaxf(1.0f - s.mass, 0.0f);
            g.mass = s.mass + q_rest;
            g.out_log = s.all + s.log_rest;
            g.out = g.mass * expf(s.log_rest) - q_rest;
        }
    }
    return g;
}
// the gradient of a class among the ids, times `mul`
__device__ __forceinline__ float own_grad(const RowGrad& g, const DsArgs& a, float at, float taken, float mul) {
    return (expf((at - g.m) * a.scale - g.all) * g.mass - taken) * mul;
}

// Loss and sums of a row from what a pass over it found, `pass`: the sum over all classes, or (TAIL) over those outside the ids,
// `own` being the sum over those (about own.m).  term: sum of q (log q - (x[id] - base) scale).  used: some slot of the row is.
template <bool TAIL>
__device__ __forceinline__ RowSums finish_row(const DsArgs& a, const RowStat& pass, const RowStat& own, float base, float term, const Teacher& t,
                                              bool used, float& loss) {
    const RowStat all = TAIL ? merge_stat<false>(pass, own, a.c) : pass;
    const float log_s = logf(all.s);
    loss = term;
    // (base is the largest logit of the ids, so that the distance is not negative; if all of them are at -inf it is 0, term is +inf,
    // and a distance below 0, down to -inf by the scale, must not take that back)
    if (t.mass != 0.0f) loss = loss + t.mass * (fmaxf((all.m - base) * a.scale, 0.0f) + log_s);
    RowSums s{all.m, log_s, -INFINITY, t.mass};
    if (TAIL && !(pass.m == -INFINITY && pass.s == 0.0f)) {
        s.log_rest = (pass.m - all.m) * a.scale + (logf(pass.s) - log_s);
        if (s.log_rest == -INFINITY) s.log_rest = -3.4028234663852886e38f;          // (there are classes outside)
        const float q_rest = fmaxf(1.0f - t.mass, 0.0f);
        if (q_rest > 0.0f) loss = loss + q_rest * (logf(q_rest) - s.log_rest);
    }
    if (!used || t.log_sum == INFINITY || (all.m == -INFINITY && all.s == 0.0f)) {
        loss = 0.0f;
        s = RowSums{-INFINITY, 0.0f, -INFINITY, 0.0f};
    } else if (log_s != log_s || !(t.mass < INFINITY)) {           // NaN or +inf among the logits, or the teacher's values
        loss = NAN;
        s = RowSums{NAN, NAN, NAN, NAN};
    }
    return s;
}
// the ids' side of that: the sum over their classes (each once), base and term
template <int BLOCK, bool TAIL>
__device__ __forceinline__ RowStat ids_side(const DsArgs& a, const Teacher& t, int32_t id, float q, float at, bool first, float& base, float& term,
                                            float* lds) {
    const float top = block_largest<BLOCK>(id >= 0 ? at : -INFINITY, lds);
    base = fabsf(top) < INFINITY ? top : 0.0f;
    float some = 0.0f, share = 0.0f;
    if (id >= 0 && !(q == 0.0f)) some = q * (t.log_q - (at - base) * a.scale);
    if (TAIL && first) share = __builtin_amdgcn_exp2f((at - base) * a.c);       // (-inf: 0)
    term = block_total<BLOCK>(some, lds);
    return RowStat{top, TAIL ? block_total<BLOCK>(share, lds) : 0.0f, 0.0f};
}

// ---- forward: a workgroup a row, or a part of one ----------------------------------------------------------
// One pass, as the log probabilities' (8192 rows of 151936 bf16 with 64 slots and a tail 383 us, 6.5 TB/s; 512 rows of 32768 fp32
// 15 us; one row of 32768 with 64 slots 7 us).
// WORDS: of the bit map, 0 in RENORM.  (A map for the longest part costs a CU its eighth workgroup, which 2048 rows of 50257 bf16
// classes feel: 46 against 41 us.)
template <typename T, int VEC, uint32_t WORDS, int BLOCK>
__global__ void __launch_bounds__(BLOCK)
distill_fwd_kernel(const T* __restrict__ x, const DsArgs a, const DsOut o) {
    constexpr bool TAIL = WORDS != 0;
    __shared__ __align__(16) uint32_t map[TAIL ? WORDS : 4];
    __shared__ uint32_t outside;
    __shared__ Slots slots;
    __shared__ float lds[BLOCK / kWave];
    __shared__ RowStat lds_stat[BLOCK / kWave];
    __shared__ uint32_t word;
    typedef RawVec<T, VEC> Raw;
    const uint32_t row = blockIdx.x / o.parts, nth = blockIdx.x - row * o.parts, k = threadIdx.x;
    const T* base = x + row * a.ld;
    const RowParts<T, VEC> parts(base, a.V);
    const Stretch part(parts.nvec, nth, o.parts);
    const T* body = base + parts.head;
    // a slot's class and value, then the first vectors, then the slot's logit: the teacher's side is done while they come
    const uint64_t slot_at = (uint64_t)row * a.top + (k < a.top ? k : 0u);
    const int32_t asked = a.ids[slot_at];
    const float given = a.values[slot_at];
    typename Raw::type raw[kDsUnroll];
    const uint32_t length = part.hi - part.lo, skew = line_skew<VEC>(body + (uint64_t)part.lo * VEC, length, BLOCK * kDsUnroll);
    auto read = [&](uint32_t i0) {
#pragma unroll
        for (int u = 0; u < kDsUnroll; ++u) {
            const uint32_t i = i0 + u * BLOCK - skew;
            raw[u] = Raw::load(body + (uint64_t)(part.lo + (i < length ? i : 0u)) * VEC);
        }
    };
    uint32_t i0 = k;
    if (i0 < length + skew) read(i0);
    const int32_t id = k < a.top && asked >= 0 && (uint32_t)asked < a.V ? asked : -1;
    if (nth == 0 && k < a.top && id != asked && asked != -1) *a.err_flag = 1;
    float at[1];
    VecIO<T, 1>::load(base + (id >= 0 ? id : 0), at);
    if (k < AGRAD_MAX_TOP) slots.id[k] = id;
    const uint32_t classes = length * VEC;
    if (TAIL) clear_map<BLOCK>(map, classes);
    if (TAIL && k == 0) outside = 0u;
    const bool used = __syncthreads_or(id >= 0) != 0;
    if (TAIL) mark(map, outside, parts, id, parts.head + part.lo * VEC, classes);
    const Teacher teach = teacher_row<BLOCK, TAIL>(a, id >= 0 ? given : -INFINITY, lds);
    const float q = expf(teach.log_q);
    const bool first = TAIL && k < AGRAD_MAX_TOP && own_slot<false>(slots, a.top, k, id).first;
    __syncthreads();
    RowStat t = empty_stat();
    while (i0 < length + skew) {
#pragma unroll
        for (int u = 0; u < kDsUnroll; ++u) {
            const uint32_t i = i0 + u * BLOCK - skew;
            if (i >= length) continue;
            if (TAIL) {
                const uint32_t bits = bits_of<VEC>(map, i);
                if (bits != 0) mask_raw(raw[u], bits);
            }
            float v[VEC];
            Raw::unpack(raw[u], v);
            absorb_stat<false, VEC>(t, v, a.c);
        }
        i0 += BLOCK * kDsUnroll;
        if (i0 < length + skew) read(i0);
    }
    if (nth == 0 && k < parts.extra) {
        const uint32_t e = parts.extra_at(k);
        float v[1];
        VecIO<T, 1>::load(base + e, v);
        if (TAIL && (outside >> k & 1u)) v[0] = -INFINITY;
        absorb_stat<false, 1>(t, v, a.c);
    }
    t = block_stat<BLOCK, false>(t, a.c, lds_stat);
    if constexpr (BLOCK == kDsBlock) if (o.parts > 1) {
        if (k == 0) {
            float* to = o.shared.stats + 4 * (uint64_t)blockIdx.x;
            put_shared(to, t.m);
            put_shared(to + 1, t.s);
        }
        if (!workgroup_arrives_last(o.shared.tickets + row, o.parts, &word)) return;
        t = empty_stat();
        if (k < o.parts) {
            const float* from = o.shared.stats + 4 * ((uint64_t)row * o.parts + k);
            t = RowStat{get_shared(from), get_shared(from + 1), 0.0f};
        }
        t = block_stat<BLOCK, false>(t, a.c, lds_stat);
    }
    float base_own, term, loss;
    const RowStat own = ids_side<BLOCK, TAIL>(a, teach, id, q, at[0], first, base_own, term, lds);
    const RowSums s = finish_row<TAIL>(a, t, own, base_own, term, teach, used, loss);
    if (k == 0) {
        if (o.loss != nullptr) o.loss[row] = loss;
        if (o.stats != nullptr) {
            float* to = o.stats + row * 4ull;
            to[0] = s.m; to[1] = s.all; to[2] = TAIL ? s.log_rest : teach.log_sum; to[3] = TAIL ? s.mass : teach.top;
            if (TAIL && s.log_rest < kFarRest && s.log_rest > -INFINITY) { to[2] = t.m; to[3] = -1.0f - logf(t.s); }
        }
    }
}

// ---- backward ----------------------------------------------------------------------------------------------
template <typename T, int VEC>
__device__ __forceinline__ void ds_store(T* to, float (&d)[VEC], uint32_t accumulate) {
    if (accumulate) {
        float old[VEC];
        VecIO<T, VEC>::load(to, old);
#pragma unroll
        for (int k = 0; k < VEC; ++k) d[k] = old[k] + d[k];
    }
    store_grad<T, VEC>(to, d);
}

// A wave takes 128 neighbouring vectors of a row, two a lane, and needs no other: it looks through the row's ids for those of its
// classes, writes its vectors as if there were none, and stores over them, each by the lane that stored its vector (in
// order).  Two vectors a lane halve the looking: 8192 rows of 32768 bf16 with 64 ids 195 us, of 8192 with 20 ids 50 us (one
// vector: 210, 57; 8192 rows of 151936 with 64 ids are 861 and 839).  A workgroup that collected the ids of its 16 KB in LDS took
// a fifth longer.
constexpr int kBwdVectors = 2;
template <int CLASSES>
struct WaveSlots {
    PatchLists<kWave> patches;
    uint32_t seen[CLASSES / 32 + 1];
};
// LDS instructions of a wave are carried out in their order; this keeps the compiler to it too
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
template <typename T, int VEC, bool TAIL>
__global__ void __launch_bounds__(kDsBlock)
distill_bwd_kernel(const T* x, T* dx, const DsArgs a, const float* dloss, const float* row_scale, float grad_scale, const float* stats,
                   uint32_t accumulate, const FastDiv32 chunks, uint32_t waves) {
    typedef RawVec<T, VEC> Raw;
    constexpr int U = kBwdVectors;
    __shared__ WaveSlots<kWave * U * VEC> lists[kDsBlock / kWave];
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t wave = blockIdx.x * (kDsBlock / kWave) + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
    if (wave >= waves) return;
    const uint32_t row = chunks.div(wave), chunk = wave - row * chunks.d;
    const T* base = x + (uint64_t)row * a.ld;
    T* out = dx + (uint64_t)row * a.ld;
    const RowParts<T, VEC> parts(base, a.V);
    // (its vectors are lo .. lo + span; of the first wave the first ones are before the row, large numbers)
    constexpr uint32_t span = kWave * U;
    const uint32_t lo = chunk * span - line_skew<VEC>(base + parts.head);
    // slots lane and lane + 64
    static_assert(AGRAD_MAX_TOP == 2 * kWave, "");
    const int32_t* ids = a.ids + (uint64_t)row * a.top;
    const int32_t id0 = lane < a.top ? ids[lane] : -1, id1 = lane + kWave < a.top ? ids[lane + kWave] : -1;
    typename Raw::type raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t i = lo + u * kWave + lane;
        raw[u] = Raw::load(base + parts.head + (uint64_t)(i < parts.nvec ? i : 0u) * VEC);
    }
    const uint32_t extra = chunk == 0 ? parts.extra : 0u, e = parts.extra_at(lane);
    float xe[1];
    VecIO<T, 1>::load(base + (lane < extra ? e : 0u), xe);
    const float* st = stats + (uint64_t)row * 4;
    RowGrad g = row_grad<TAIL>(RowSums{st[0], st[1], TAIL ? st[2] : -INFINITY, TAIL ? st[3] : 1.0f});
    float from = g.m;                                     // what the exponentials of the classes outside are about
    if (TAIL && st[3] < 0.0f) {
        auto q_of = [&](int32_t id, uint32_t slot) { return id >= 0 && (uint32_t)id < a.V ? expf(a.values[(uint64_t)row * a.top + slot]) : 0.0f; };
        const float mass = wave_sum(q_of(id0, lane) + q_of(id1, lane + kWave)), q_rest = fmaxf(1.0f - mass, 0.0f);
        from = st[2];
        g.out_log = -1.0f - st[3];
        g.out = -q_rest;
        g.mass = mass + q_rest;
    }
    const float mul = a.scale * (dloss != nullptr ? dloss[row] : row_scale != nullptr ? row_scale[row] : grad_scale);
    const bool none = g.m == -INFINITY;

    // who stores the class, if this wave does
    auto owner = [&](int32_t id) {
        const uint32_t v = (uint32_t)id;
        if (id < 0 || v >= a.V) return 0xffffffffu;
        const uint32_t vec = v >= parts.head ? (v - parts.head) / VEC : 0xffffffffu;
        if (vec < parts.nvec) return vec - lo < span ? (vec - lo) % kWave : 0xffffffffu;
        return chunk == 0 ? (v < parts.head ? v : parts.head + (v - parts.tail_start)) : 0xffffffffu;
    };
    if (chunk == 0 && dloss != nullptr && ((id0 != -1 && (uint32_t)id0 >= a.V) || (id1 != -1 && (uint32_t)id1 >= a.V))) *a.err_flag = 1;
    const uint32_t who0 = none ? 0xffffffffu : owner(id0), who1 = none ? 0xffffffffu : owner(id1);
    const uint64_t mine0 = __ballot(who0 != 0xffffffffu), mine1 = __ballot(who1 != 0xffffffffu);
    float at0[1] = {0.0f}, at1[1] = {0.0f}, old0[1] = {0.0f}, old1[1] = {0.0f}, q0 = 0.0f, q1 = 0.0f;
    if ((mine0 | mine1) != 0) {
        auto ask = [&](bool has, int32_t id, uint32_t slot, float (&at)[1], float (&old)[1], float& q) {
            if (!has) return;
            const float u = a.values[(uint64_t)row * a.top + slot];
            VecIO<T, 1>::load(base + id, at);
            if (accumulate) VecIO<T, 1>::load(out + id, old);
            q = expf(TAIL ? u : renorm_log_q(u, st[3], st[2], a.teacher_scale));
        };
        ask(who0 != 0xffffffffu, id0, lane, at0, old0, q0);
        ask(who1 != 0xffffffffu, id1, lane + kWave, at1, old1, q1);
    }

    const float k = none ? 0.0f : g.out * mul, b = -g.out_log * kLog2eHi;
    if (none && accumulate) return;
    if (lane < extra) {
        float d[1] = {none ? 0.0f : __builtin_amdgcn_exp2f(__builtin_fmaf(xe[0] - from, a.c, b)) * k};
        ds_store<T, 1>(out + e, d, accumulate);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t i = lo + u * kWave + lane;
        if (i >= parts.nvec) continue;
        float v[VEC];
        Raw::unpack(raw[u], v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = none ? 0.0f : __builtin_amdgcn_exp2f(__builtin_fmaf(v[j] - from, a.c, b)) * k;
        ds_store<T, VEC>(out + parts.head + (uint64_t)i * VEC, v, accumulate);
    }
    if ((mine0 | mine1) == 0) return;
    // A class that the row names twice counts with both its q and is stored for its first slot: slots whose bit is there already
    // have the wave look for such classes, which otherwise has nothing to compare.
    auto& w = lists[threadIdx.x / kWave];
    w.patches.head[lane] = w.patches.kNone;
    if (lane < sizeof(w.seen) / 4) w.seen[lane] = 0u;
    wave_lds_order();
    auto seen = [&](bool has, int32_t id, uint32_t who) {
        const uint32_t v = (uint32_t)id - parts.head - lo * VEC;                // (outside the vectors: the bits behind theirs)
        const uint32_t bit = (uint32_t)id >= parts.head && (uint32_t)id < parts.tail_start ? v : span * VEC + who;
        return has && (atomicOr(&w.seen[bit / 32], 1u << (bit % 32)) >> (bit % 32) & 1u) != 0;
    };
    bool first0 = who0 != 0xffffffffu, first1 = who1 != 0xffffffffu;
    float taken0 = q0, taken1 = q1;
    const bool again0 = seen(first0, id0, who0), again1 = seen(first1, id1, who1);
    if (__ballot(again0 || again1) != 0) {
        auto of_lane = [](float v, int l) { return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), l)); };
        auto gather = [&](uint64_t these, int32_t id, bool upper) {
            for (; these != 0; these &= these - 1) {
                const int l = (int)__builtin_ctzll(these);
                const int32_t which = __builtin_amdgcn_readlane(id, l);
                const uint64_t same0 = __ballot(id0 == which), same1 = __ballot(id1 == which);
                float taken = 0.0f;
                for (uint64_t m = same0; m != 0; m &= m - 1) taken = taken + of_lane(q0, (int)__builtin_ctzll(m));
                for (uint64_t m = same1; m != 0; m &= m - 1) taken = taken + of_lane(q1, (int)__builtin_ctzll(m));
                const bool first = upper ? same0 == 0 && (int)__builtin_ctzll(same1) == l : (int)__builtin_ctzll(same0) == l;
                const bool me = lane == (uint32_t)l;
                if (upper) { taken1 = me ? taken : taken1; first1 = me ? first : first1; }
                else { taken0 = me ? taken : taken0; first0 = me ? first : first0; }
            }
        };
        gather(mine0, id0, false);
        gather(mine1, id1, true);
    }
    if (first0) w.patches.add(lane, who0, id0, own_grad(g, a, at0[0], taken0, mul) + old0[0]);
    if (first1) w.patches.add(lane + kWave, who1, id1, own_grad(g, a, at1[0], taken1, mul) + old1[0]);
    wave_lds_order();
    w.patches.store(out, lane);
}

// ---- loss and gradient in one launch, the row in registers in between ------------------------------------------
// A workgroup a row, which it holds in registers between the sums and the gradient: 20 vectors a thread leave two 512-thread
// workgroups to a CU, longer rows of fp32 take one of 1024 threads.  Sums are taken in the order of the loads, with the running
// maximum of each thread, while later vectors are on their way; what a row needs besides its vectors is asked for before
// them (waits are in order: behind them it would wait for the whole row).  The classes among the ids are stored a second time, by
// the thread that stored their vector: in order, without a wait for the stores.  x and dx may be the same memory.  8192 rows of
// 32768 fp32 with 32 slots 385 us, 5.6 TB/s of what is read and written.
// (Workgroups that stay and ask for their next row's vectors as they store this one's were slower by 4 to 20 %, with no
// register spilled: 424 against 400 us for 8192 rows of 32768 fp32.)
// With NV = 0 the row is read twice instead: the first pass reads with ordinary loads, which leave the rows that are being worked
// on (one or two a CU, some 100 to 260 MB) in the memory-side cache, the second with loads that pass by it.  (Reading and writing
// 2048 rows of 128256 fp32 like this takes a kernel without arithmetic 432 us, with both passes passing by the cache 583; this one
// 450, and 8192 rows of 151936 bf16 1025.)
template <typename T, int VEC, int NV, int BLOCK, bool TAIL>
__global__ void __launch_bounds__(BLOCK, NV == 0 ? 8 : 1)
distill_held_kernel(const T* x, T* dx, const DsArgs a, const DsOut o) {
    constexpr int U = NV != 0 ? NV : kDsUnroll;                   // vectors a thread has in registers
    __shared__ __align__(16) uint32_t map[!TAIL ? 4 : NV != 0 ? NV * BLOCK * VEC / 32 : kMapWords];
    __shared__ uint32_t outside;
    __shared__ Slots slots;
    __shared__ PatchLists<BLOCK> patches;
    __shared__ float lds[BLOCK / kWave];
    __shared__ RowStat lds_stat[BLOCK / kWave];
    typedef RawVec<T, VEC> Raw;
    const uint32_t tid = threadIdx.x, row = blockIdx.x;
    const T* base = x + (uint64_t)row * a.ld;
    T* out = dx + (uint64_t)row * a.ld;
    const RowParts<T, VEC> parts(base, a.V);
    // a slot's class and value, an element outside the vectors; then the row; then the slot's logit
    const uint64_t slot_at = (uint64_t)row * a.top + (tid < a.top ? tid : 0u);
    const int32_t asked = a.ids[slot_at];
    const float given = a.values[slot_at];
    float at[1], xe[1];
    VecIO<T, 1>::load(base + (tid < parts.extra ? parts.extra_at(tid) : 0u), xe);
    typename Raw::type raw[U];
    // places of vectors count from the 128 bytes in which the first one lies
    const uint32_t skew = line_skew<VEC>(base + parts.head, parts.nvec, U * BLOCK), places = parts.nvec + skew;
    auto read = [&](uint32_t from) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const uint32_t vec = from + (uint32_t)i * BLOCK + tid - skew;
            const T* at_ = base + parts.head + (uint64_t)(vec < parts.nvec ? vec : 0u) * VEC;
            if constexpr (NV != 0) raw[i] = Raw::load(at_);
            else raw[i] = *reinterpret_cast<const typename Raw::type*>(at_);
        }
    };
    read(0);
    if (TAIL) clear_map<BLOCK>(map, NV != 0 ? (uint32_t)(NV * BLOCK * VEC) : places * VEC);
    if (TAIL && tid == 0) outside = 0u;
    patches.head[tid] = patches.kNone;
    const int32_t id = tid < a.top && asked >= 0 && (uint32_t)asked < a.V ? asked : -1;
    if (tid < a.top && id != asked && asked != -1) *a.err_flag = 1;
    const float u = id >= 0 ? given : -INFINITY;
    VecIO<T, 1>::load(base + (id >= 0 ? id : 0), at);
    const bool used = __syncthreads_or(id >= 0) != 0;

    // the teacher's side, and what the student says of the ids' classes
    if (tid < AGRAD_MAX_TOP) slots.id[tid] = id;
    if (TAIL) mark(map, outside, parts, id, parts.head - skew * VEC, places * VEC);
    const Teacher teach = teacher_row<BLOCK, TAIL>(a, u, lds);
    const float q = expf(teach.log_q);
    if (tid < AGRAD_MAX_TOP) slots.q[tid] = q;
    __syncthreads();
    const Own own = own_slot<true>(slots, a.top, tid, id);
    if (TAIL && (outside >> (tid % 32) & 1u)) xe[0] = -INFINITY;       // (at most 15 of them; the others' are not looked at)
    if (tid >= parts.extra) xe[0] = -INFINITY;

    RowStat t = empty_stat();
    absorb_stat<false, 1>(t, xe, a.c);
    // (with NV the map covers all vectors of a thread; a step of BLOCK vectors is whole words)
    static_assert(BLOCK * VEC % 32 == 0, "");
    const uint32_t shift_bits = tid * VEC % 32;
    for (uint32_t from = 0; from < places; from += U * BLOCK) {
        if (NV == 0 && from != 0) read(from);
        const uint32_t* words = map + (TAIL ? (from + tid) * VEC / 32 : 0u);
        uint32_t bits = TAIL && from + tid < places ? words[0] : 0u;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const uint32_t place = from + (uint32_t)i * BLOCK + tid;
            uint32_t ahead = 0;
            if (TAIL && i + 1 < U && (NV != 0 || place + BLOCK < places)) {
                ahead = words[(i + 1) * (BLOCK * VEC / 32)];
                asm volatile("" ::: "memory");                     // (one vector's bits ahead, not all of them)
            }
            if (place - skew < parts.nvec) {
                if (TAIL) {
                    bits = (bits >> shift_bits) & ((1u << VEC) - 1u);
                    if (bits != 0) mask_raw(raw[i], bits);
                }
                float v[VEC];
                Raw::unpack(raw[i], v);
                absorb_stat<false, VEC>(t, v, a.c);
            }
            if constexpr (NV != 0) unpack_again(raw[i]);
            bits = ahead;
        }
        if constexpr (NV != 0) break;
    }
    t = block_stat<BLOCK, false>(t, a.c, lds_stat);

    float about_own, term, loss;
    const RowStat own_sum = ids_side<BLOCK, TAIL>(a, teach, id, q, at[0], own.first, about_own, term, lds);
    const RowSums s = finish_row<TAIL>(a, t, own_sum, about_own, term, teach, used, loss);
    if (tid == 0 && o.loss != nullptr) o.loss[row] = loss;
    const RowGrad g = row_grad<TAIL>(s);
    const float mul = a.scale * (o.row_scale != nullptr ? o.row_scale[row] : o.grad_scale);
    if (g.m == -INFINITY) {                                         // (no gradient: zeros, whatever the logits hold)
        float v[VEC] = {};
        float d[1] = {0.0f};
        if (tid < parts.extra) VecIO<T, 1>::store(out + parts.extra_at(tid), d);
        for (uint32_t vec = tid; vec < parts.nvec; vec += BLOCK) VecIO<T, VEC>::store(out + parts.head + (uint64_t)vec * VEC, v);
        return;
    }
    // hand the ids' gradients to the threads that store their vectors
    if (own.first) {
        const uint32_t vec = (uint32_t)id >= parts.head ? ((uint32_t)id - parts.head) / VEC : 0xffffffffu;
        const uint32_t who = vec < parts.nvec ? (vec + skew) % BLOCK : ((uint32_t)id < parts.head ? (uint32_t)id : parts.head + ((uint32_t)id - parts.tail_start));
        patches.add(tid, who, id, own_grad(g, a, at[0], own.taken, mul));
    }
    __syncthreads();

    // exponentials about the largest logit outside the ids (RENORM: of all)
    const float shift = t.m > -INFINITY ? t.m : 0.0f;
    const float k = g.out * mul / (t.s == 0.0f ? 1.0f : t.s);            // (without classes outside g.out is 0, or NaN with the row)
    if (tid < parts.extra) {
        float d[1] = {__builtin_amdgcn_exp2f((xe[0] - shift) * a.c) * k};
        VecIO<T, 1>::store(out + parts.extra_at(tid), d);
    }
    // (the thread's number is read anew: what the compiler would keep of it, an index and an address a vector, costs the
    // longest rows their last registers)
    uint32_t again = tid;
    asm volatile("" : "+v"(again));
    auto rewrite = [&](const typename Raw::type& r, uint32_t vec) {
        float v[VEC];
        Raw::unpack(r, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = __builtin_amdgcn_exp2f((v[j] - shift) * a.c) * k;
        if (vec < parts.nvec) store_grad<T, VEC>(out + parts.head + (uint64_t)vec * VEC, v);
    };
    if constexpr (NV != 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) rewrite(raw[i], (uint32_t)i * BLOCK + again - skew);
    } else {
        for (uint32_t from = again; from < places; from += 2 * BLOCK) {
            typename Raw::type two[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t vec = from + (uint32_t)i * BLOCK - skew;
                two[i] = Raw::load(base + parts.head + (uint64_t)(vec < parts.nvec ? vec : 0u) * VEC);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) rewrite(two[i], from + (uint32_t)i * BLOCK - skew);
        }
    }
    patches.store(out, tid);
}

inline bool one_alignment(const void* x, const void* dx) {
    return ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15u) == 0;
}

template <typename T>
int ds_fwd_typed(hipStream_t s, const T* x, const DsArgs& a, DsOut o, uint64_t rows, bool tail) {
    constexpr int WIDE = WideVec<T>::value;
    const bool wide = a.V >= 4 * WIDE;
    const uint32_t vectors = wide ? a.V / WIDE : a.V;
    o.parts = wide ? row_parts(rows, vectors) : 1u;
    uint64_t slab = rows;
    if (tail && (vectors + o.parts - 1) / o.parts > kMapBits / WIDE) {
        // a part's classes have to fit the bit map: rows longer than it are cut, so many rows a launch as the parts' memory takes
        o.parts = (vectors + kMapBits / WIDE - 1) / (kMapBits / WIDE);             // (at most kMaxParts: the classes are checked)
        slab = kSharedParts / o.parts;
    }
    const uint32_t longest = ((vectors + o.parts - 1) / o.parts) * (wide ? WIDE : 1);        // classes of a part's vectors, at most
    for (uint64_t r0 = 0; r0 < rows; r0 += slab) {
        const uint64_t n = rows - r0 < slab ? rows - r0 : slab;
        DsArgs b = a;
        DsOut p = o;
        b.ids += r0 * a.top;
        b.values += r0 * a.top;
        if (p.loss) p.loss += r0;
        if (p.stats) p.stats += 4 * r0;
        const dim3 grid((uint32_t)n * o.parts);
        const T* from = x + r0 * a.ld;
#define AGRAD_DS(VEC, WORDS, BLOCK) hipLaunchKernelGGL((distill_fwd_kernel<T, VEC, WORDS, BLOCK>), grid, dim3(BLOCK), 0, s, from, b, p)
        // (short rows as below: 32768 of 257 fp32 with 10 slots 19 us in 64 threads, 37 in 128, 71 in 256)
        if (wide && o.parts == 1 && longest <= 128u * kDsUnroll * WIDE) {
            if (a.top <= 64 && longest <= 64u * kDsUnroll * WIDE) {
                if (tail) AGRAD_DS(WIDE, 64 * kDsUnroll * WIDE / 32, 64); else AGRAD_DS(WIDE, 0, 64);
            }
            else if (tail) AGRAD_DS(WIDE, 128 * kDsUnroll * WIDE / 32, 128); else AGRAD_DS(WIDE, 0, 128);
        } else if (wide && tail && longest <= kShortMap * 32) AGRAD_DS(WIDE, kShortMap, kDsBlock);
        else if (wide && tail) AGRAD_DS(WIDE, kMapWords, kDsBlock);
        else if (wide) AGRAD_DS(WIDE, 0, kDsBlock);
        else if (tail) AGRAD_DS(1, kShortMap, kDsBlock);
        else AGRAD_DS(1, 0, kDsBlock);
#undef AGRAD_DS
    }
    return check_hip(hipGetLastError(), "top-k distillation launch");
}

template <typename T>
int ds_bwd_typed(hipStream_t s, const T* x, T* dx, const DsArgs& a, const float* dloss, const float* row_scale, float grad_scale,
                 const float* stats, uint32_t accumulate, uint64_t rows, bool tail) {
    constexpr int WIDE = WideVec<T>::value;
    const bool wide = a.V >= 4 * WIDE && one_alignment(x, dx);
    const uint32_t vec = wide ? WIDE : 1, span = kWave * kBwdVectors;
    const bool lines = ((reinterpret_cast<uintptr_t>(x) | (rows > 1 ? a.ld * sizeof(T) : 0u)) & 127u) == 0;      // every row at 128 bytes
    const uint32_t chunks = (a.V / vec + (wide && !lines ? 7u : 0u) + span - 1) / span;
    uint64_t max_rows = 0x03ffffffull / chunks;                  // waves of a launch: 2^32 threads
    if (max_rows == 0) max_rows = 1;
    for (uint64_t r0 = 0; r0 < rows; r0 += max_rows) {
        const uint64_t n = rows - r0 < max_rows ? rows - r0 : max_rows;
        DsArgs b = a;
        b.ids += r0 * a.top;
        b.values += r0 * a.top;
        const uint32_t waves = (uint32_t)(n * chunks);
        const dim3 grid((waves + kDsBlock / kWave - 1) / (kDsBlock / kWave)), block(kDsBlock);
#define AGRAD_DS(VEC, TAIL) hipLaunchKernelGGL((distill_bwd_kernel<T, VEC, TAIL>), grid, block, 0, s, x + r0 * a.ld, dx + r0 * a.ld, b, dloss ? dloss + r0 : nullptr, row_scale ? row_scale + r0 : nullptr, grad_scale, stats + 4 * r0, accumulate, FastDiv32(chunks), waves)
        if (wide) { if (tail) AGRAD_DS(WIDE, true); else AGRAD_DS(WIDE, false); }
        else if (tail) AGRAD_DS(1, true);
        else AGRAD_DS(1, false);
#undef AGRAD_DS
    }
    return check_hip(hipGetLastError(), "top-k distillation backward launch");
}

template <typename T, bool TAIL>
bool ds_held_launch(hipStream_t s, const T* x, T* dx, const DsArgs& a, const DsOut& o, uint64_t rows) {
    constexpr int WIDE = WideVec<T>::value;
    const uint32_t vectors = a.V / WIDE;
    const dim3 grid((uint32_t)rows);
    // Held rows of two 512-thread workgroups a CU are faster than rows read twice (2048 x 50257 bf16 82 against 95 us, 4096 x 20000 70
    // against 94, 8192 x 32768 fp32 386 against 419).  Beyond them a CU holds 1024 threads at a time: fp32 still gains or is even (4096 x
    // 80000 514 against 548 us, 4096 x 50257 346 against 351, 512 x 70000 65 in both), bf16, with twice the arithmetic a byte and no
    // second workgroup to fill its waits, loses (1024 x 110000 120 against 102 us, 8192 x 151936 1130 against 1075).
#define AGRAD_DS(N, BLOCK) \
    if (vectors <= (uint32_t)(N) * BLOCK) { hipLaunchKernelGGL((distill_held_kernel<T, WIDE, N, BLOCK, TAIL>), grid, dim3(BLOCK), 0, s, x, dx, a, o); return true; }
    // Short rows take the smallest workgroup that has four vectors a thread and a thread a slot, as the reductions of its waves are
    // most of their time (32768 rows of 257 fp32: 10 slots 26 us in 64 threads, 46 in 128, 83 in 256; 100 slots 84 in 128, 137 in
    // 256; 8192 rows of 4000 bf16, 10 slots: 28 in 128, 36 in 256).
    if (a.top <= 64) { AGRAD_DS(2, 64) AGRAD_DS(4, 64) }
    AGRAD_DS(2, 128) AGRAD_DS(4, 128) AGRAD_DS(4, 256) AGRAD_DS(4, 512) AGRAD_DS(8, 512) AGRAD_DS(12, 512) AGRAD_DS(16, 512) AGRAD_DS(20, 512)
    if constexpr (sizeof(T) == 4) {
        AGRAD_DS(12, 1024) AGRAD_DS(16, 1024) AGRAD_DS(20, 1024)
    }
#undef AGRAD_DS
    if (TAIL && vectors + 8 > kMapBits / WIDE) return false;
    hipLaunchKernelGGL((distill_held_kernel<T, WIDE, 0, 1024, TAIL>), grid, dim3(1024), 0, s, x, dx, a, o);
    return true;
}

// A few long rows, rows with a tail whose ids' bit map is more than LDS, rows of a few classes, and logits and gradient at different
// places within 16 bytes: the forward pass, then the backward pass, over as many rows at a time as the context's memory holds sums for.
template <typename T>
int ds_fused_typed(hipStream_t s, const T* x, T* dx, const DsArgs& a, const DsOut& o, uint64_t rows, bool tail) {
    constexpr int WIDE = WideVec<T>::value;
    // A CU takes up to 25 us for a long row; few of them are faster shared out in two launches, which are faster up to some number of rows
    // that grows with the classes beyond 6000 vectors: one row of 151936 bf16 10.9 against 24.4 us, 96 rows 27.7 against 28.3, 160
    // rows 36.9 against 33.7; of 90000 bf16, 32 rows 14.9 against 18.0, 64 rows 18.3 against 18.1; of 60000 fp32, 32 rows 14.8
    // against 15.1, 64 rows 19.1 against 16.0; of 40000, 8 rows 11.2 against 11.5, 32 rows 13.2 against 11.9; of 32768 bf16, one
    // row 10.8 against 9.3.
    const bool few = a.V > 6000 * WIDE && rows * 900 <= a.V - 6000 * WIDE;
    if (a.V >= 4 * WIDE && one_alignment(x, dx) && !few) {
        if (tail ? ds_held_launch<T, true>(s, x, dx, a, o, rows) : ds_held_launch<T, false>(s, x, dx, a, o, rows))
            return check_hip(hipGetLastError(), "top-k distillation step launch");
    }
    for (uint64_t r0 = 0; r0 < rows; r0 += kSumRows) {
        const uint64_t n = rows - r0 < kSumRows ? rows - r0 : kSumRows;
        DsArgs b = a;
        DsOut p = o;
        b.ids += r0 * a.top;
        b.values += r0 * a.top;
        if (p.loss) p.loss += r0;
        p.stats = o.shared.sums;
        if (int rc = ds_fwd_typed<T>(s, x + r0 * a.ld, b, p, n, tail)) return rc;
        if (int rc = ds_bwd_typed<T>(s, x + r0 * a.ld, dx + r0 * a.ld, b, nullptr, o.row_scale ? o.row_scale + r0 : nullptr, o.grad_scale,
                                     o.shared.sums, 0u, n, tail)) return rc;
    }
    return AGRAD_OK;
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
    if (mode == AGRAD_DISTILL_TAIL && V > AGRAD_MAX_TAIL_CLASSES)
        return set_error(AGRAD_EINVAL, "%s: %u classes, at most %u with a tail", what, V, AGRAD_MAX_TAIL_CLASSES);
    if (rows != 0 && (logits == nullptr || ids == nullptr || values == nullptr)) return set_error(AGRAD_EINVAL, "%s: null operand", what);
    const float c = (float)((double)scale * 1.4426950408889634);
    *a = DsArgs{ids, values, ld, V, top, scale, c, teacher_scale, err_flag};
    return AGRAD_OK;
}

}  // namespace

int launch_distill_fwd(hipStream_t s, int dtype, const void* logits, const int32_t* ids, const float* values, float* loss, float* stats,
                       uint64_t rows, uint32_t V, uint64_t ld, uint32_t top, float scale, float teacher_scale, int mode, int* err_flag,
                       void* scratch) {
    DsArgs a;
    if (int rc = ds_args("top-k distillation", dtype, logits, ids, values, nullptr, rows, V, ld, top, scale, teacher_scale, mode, err_flag, &a)) return rc;
    if (rows == 0) return AGRAD_OK;
    if (loss == nullptr) return set_error(AGRAD_EINVAL, "top-k distillation: null loss");
    const DsOut o{loss, stats, nullptr, 0.0f, shared_rows(scratch), 1u};
    const bool tail = mode == AGRAD_DISTILL_TAIL;
    if (dtype == AGRAD_F32) return ds_fwd_typed<float>(s, (const float*)logits, a, o, rows, tail);
    return ds_fwd_typed<bf16_t>(s, (const bf16_t*)logits, a, o, rows, tail);
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
    const bool tail = mode == AGRAD_DISTILL_TAIL;
    if (dtype == AGRAD_F32) return ds_bwd_typed<float>(s, (const float*)logits, (float*)dlogits, a, dloss, nullptr, 0.0f, stats, acc, rows, tail);
    return ds_bwd_typed<bf16_t>(s, (const bf16_t*)logits, (bf16_t*)dlogits, a, dloss, nullptr, 0.0f, stats, acc, rows, tail);
}

int launch_distill_fused(hipStream_t s, int dtype, const void* logits, const int32_t* ids, const float* values, float* loss,
                         const float* row_scale, void* dlogits, uint64_t rows, uint32_t V, uint64_t ld, uint32_t top, float scale,
                         float teacher_scale, float grad_scale, int mode, int* err_flag, void* scratch) {
    DsArgs a;
    if (int rc = ds_args("top-k distillation step", dtype, logits, ids, values, dlogits, rows, V, ld, top, scale, teacher_scale, mode, err_flag, &a)) return rc;
    if (rows == 0) return AGRAD_OK;
    if (dlogits == nullptr) return set_error(AGRAD_EINVAL, "top-k distillation step: null gradient");
    const DsOut o{loss, nullptr, row_scale, grad_scale, shared_rows(scratch), 1u};
    const bool tail = mode == AGRAD_DISTILL_TAIL;
    if (dtype == AGRAD_F32) return ds_fused_typed<float>(s, (const float*)logits, (float*)dlogits, a, o, rows, tail);
    return ds_fused_typed<bf16_t>(s, (const bf16_t*)logits, (bf16_t*)dlogits, a, o, rows, tail);
}

}  // namespace agrad
