// Losses of a policy whose action is a token of a large vocabulary: log-probability and entropy, the clipped
// surrogate with a KL term, the preference loss on pairs, distillation from a teacher's top logits, and the
// gradients of all of them with respect to the logits.
//
// Mathematics of a row (one position of one sequence), x_i its V logits, c = 1/temperature, y its token:
//   p_i = exp(c x_i - lse),  logp = c x_y - lse,  H = -sum_i p_i ln p_i
//   dL/dx_i = c (g_lp ([i = y] - p_i) - g_H p_i (ln p_i + H))          g_lp = dL/dlogp, g_H = dL/dH
// Everything a row needs of its V logits is (m, S, E) = (max x, sum e_i, sum e_i u_i) with
// u_i = (x_i - m) c log2(e), e_i = 2^u_i: lse = c m + ln S, H = ln S - ln2 E / S, p_i = e_i / S.  The three are
// kept per thread with a running maximum, joined over the workgroup, and the gradient is one multiply-add and a
// product on each e_i.  A logit of -inf or of the type's lowest value has e_i = 0.  Sums are fp32 within a thread and
// over the workgroup, one row's scalars are finished in fp64.
//
// What bounds it: memory.  With gradient a bf16 logit is 4 bytes of traffic and the time of some 16 instructions (10, of
// which two exponentials count as four each), two thirds of what the vector units can do while the memory moves it.  So a row is
// read once and stays on the chip until its gradient is written (policy_kernel, distill_kernel), or, where its gradient
// waits for other rows or a later call, is read a second time in reverse order, from the cache as far as that reaches.
// Measured, bf16, whole calls: 4096 rows of 131072 logits with gradient 5.4 TB/s of logits and gradients (a plain copy
// reaches 5.1 to 5.4), 8184 rows of 50001 forward only 6.3 TB/s (reading alone 6.1 to 6.3).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ppo_hip.h"

#define LN2_D 0.6931471805599453
#define U_FLOOR (-1.0e6f)    // below it e_i is 0: products e_i u_i take this in place of -inf

#define RED_SUM PPO_REDUCE_SUM
#define RED_TOKEN PPO_REDUCE_TOKEN_MEAN
#define RED_SEQ PPO_REDUCE_SEQUENCE_MEAN

// ------------------------------------------------------------------------------------------ element types
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Element type and how 32 bits of a row hold it; 16 bytes are kept as four words, unpacked where they are used.
template <typename T> struct Word;
template <> struct Word<float> {
    static constexpr int N = 1;
    static __device__ __forceinline__ void unpack(uint32_t w, float* f) { f[0] = __uint_as_float(w); }
    static __device__ __forceinline__ uint32_t pack(const float* f) { return __float_as_uint(f[0]); }
    static constexpr uint32_t LOWEST = 0xff800000u;    // -inf
};
template <> struct Word<__bf16> {
    static constexpr int N = 2;
    static __device__ __forceinline__ void unpack(uint32_t w, float* f) {
        f[0] = __uint_as_float(w << 16);
        f[1] = __uint_as_float(w & 0xffff0000u);
    }
    static __device__ __forceinline__ uint32_t pack(const float* f) {   // to nearest even
        const f32x2 v = {f[0], f[1]};
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
    }
    static constexpr uint32_t LOWEST = 0xff80ff80u;
};
template <> struct Word<_Float16> {
    static constexpr int N = 2;
    static __device__ __forceinline__ void unpack(uint32_t w, float* f) {
        const f16x2 h = __builtin_bit_cast(f16x2, w);
        f[0] = (float)h.x;
        f[1] = (float)h.y;
    }
    static __device__ __forceinline__ uint32_t pack(const float* f) {   // to nearest even
        const f32x2 v = {f[0], f[1]};
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
    }
    static constexpr uint32_t LOWEST = 0xfc00fc00u;
};

template <typename T> constexpr int VEC = 4 * Word<T>::N;     // elements of 16 bytes

template <typename T> __device__ __forceinline__ void unpack(u32x4 v, float* f) {
#pragma unroll
    for (int k = 0; k < 4; ++k) Word<T>::unpack(v[k], f + k * Word<T>::N);
}
template <typename T> __device__ __forceinline__ u32x4 pack(const float* f) {
    u32x4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = Word<T>::pack(f + k * Word<T>::N);
    return v;
}

__device__ __forceinline__ float wide(float x) { return x; }
__device__ __forceinline__ float wide(__bf16 x) { return (float)x; }
__device__ __forceinline__ float wide(_Float16 x) { return (float)x; }

__device__ __forceinline__ int64_t int_at(const void* p, int is_i64, int64_t i) {
    return is_i64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

__device__ __forceinline__ float float_at(const void* p, int dtype, int64_t i) {
    return dtype == PPO_F32 ? ((const float*)p)[i] : dtype == PPO_BF16 ? wide(((const __bf16*)p)[i])
                                                                       : wide(((const _Float16*)p)[i]);
}

// ------------------------------------------------------------------------------------------ row statistics
struct Acc {
    float m, s, e;
    float n;                  // counted rows of the mask, where a kernel counts them itself
};

__device__ __forceinline__ Acc acc_empty() { return {-__FLT_MAX__, 0.0f, 0.0f, 0.0f}; }   // finite: -inf logits give u = -inf

// u_i has two forms.  Exact: (x - m) c2.  NEAR: fma(x, c2, -M) with M = m c2 rounded, one instruction less for each
// logit; what M is off by, at most 2^-24 |M|, is the same for all terms of a row and is put back by near_done().  It
// needs |M| < NEAR_LIMIT: rows beyond (logits of a million and more, rows of nothing but -inf) are done over exactly.
#define NEAR_LIMIT 1048576.0f
__device__ __forceinline__ float near_max(float m, float c2) { return fmaxf(m * c2, -NEAR_LIMIT); }
__device__ __forceinline__ bool is_near(float m, float c2) { return fabsf(m * c2) < NEAR_LIMIT; }

// a, relative to a larger maximum mn
template <bool ENT, bool NEAR = false> __device__ __forceinline__ void acc_rebase(Acc& a, float mn, float c2) {
    const float d = NEAR ? near_max(a.m, c2) - near_max(mn, c2) : fmaxf((a.m - mn) * c2, -1.0e30f);
    const float r = __builtin_amdgcn_exp2f(d);
    if (ENT) a.e = fmaf(a.s, d, a.e) * r;
    a.s *= r;
    a.m = mn;
}

template <bool NEAR> __device__ __forceinline__ float u_of(float x, float m, float c2) {   // m >= x, or x is NaN
    return NEAR ? fmaf(x, c2, -near_max(m, c2)) : (x - m) * c2;
}
template <bool ENT, bool NEAR = false> __device__ __forceinline__ void acc_add(Acc& a, float x, float c2) {
    const float u = u_of<NEAR>(x, a.m, c2), e = __builtin_amdgcn_exp2f(u);
    a.s += e;
    if (ENT) a.e = fmaf(e, fmaxf(u, U_FLOOR), a.e);
}

// 16 * M bytes of logits at once: their maximum, one rescaling, their terms.  The terms are summed by themselves and then
// added: one by one the many small terms of a long row are below half a step of a sum that has grown, and S comes out
// too small (131072 normal logits of deviation 5: ln p too large by 6e-7 in the mean).
template <typename T, int M, bool ENT, bool NEAR = false>
__device__ __forceinline__ void acc_vecs(Acc& a, const u32x4* v, float c2) {
    constexpr int N = VEC<T>;
    float f[N * M], mx = a.m;
#pragma unroll
    for (int k = 0; k < M; ++k) unpack<T>(v[k], f + k * N);
#pragma unroll
    for (int i = 0; i < N * M; ++i) mx = fmaxf(mx, f[i]);
    acc_rebase<ENT, NEAR>(a, mx, c2);
    float s, e;
#pragma unroll
    for (int i = 0; i < N * M; ++i) {
        const float u = u_of<NEAR>(f[i], mx, c2), t = __builtin_amdgcn_exp2f(u);
        s = i ? s + t : t;
        if (ENT) e = i ? fmaf(t, fmaxf(u, U_FLOOR), e) : t * fmaxf(u, U_FLOOR);
    }
    a.s += s;
    if (ENT) a.e += e;
}

// The sums as they are relative to m c2 itself: with rho = m c2 - M the terms are e_i 2^-rho, u_i - rho.
__device__ __forceinline__ Acc near_done(Acc a, float c2) {
    const float rho = (float)((double)a.m * (double)c2 - (double)near_max(a.m, c2));
    const float f = __builtin_amdgcn_exp2f(-rho);
    return {a.m, a.s * f, (a.e - rho * a.s) * f, a.n};
}

// Rotation within the 16 lanes of a row: an all-reduce in four steps without LDS.  Partners add the same two
// numbers, so all lanes end with the same bits.
template <int CTRL> __device__ __forceinline__ float ror(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float lane_value(float x, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, ror<0x128>(x));
    x = fmaxf(x, ror<0x124>(x));
    x = fmaxf(x, ror<0x122>(x));
    return fmaxf(x, ror<0x121>(x));
}
__device__ __forceinline__ float row_sum(float x) {
    x += ror<0x128>(x);
    x += ror<0x124>(x);
    x += ror<0x122>(x);
    return x + ror<0x121>(x);
}
__device__ __forceinline__ float wave_max(float x) {
    x = row_max(x);
    return fmaxf(fmaxf(lane_value(x, 0), lane_value(x, 16)), fmaxf(lane_value(x, 32), lane_value(x, 48)));
}
__device__ __forceinline__ float wave_sum(float x) {
    x = row_sum(x);
    return (lane_value(x, 0) + lane_value(x, 16)) + (lane_value(x, 32) + lane_value(x, 48));
}

// The accumulators of a wave's lanes joined, the same bits in every lane.
template <bool ENT, bool NEAR = false> __device__ __forceinline__ Acc acc_wave(Acc a, float c2) {
    acc_rebase<ENT, NEAR>(a, wave_max(a.m), c2);
    a.s = wave_sum(a.s);
    if (ENT) a.e = wave_sum(a.e);
    a.n = wave_sum(a.n);
    return a;
}

// And those of the workgroup's waves (at most 16), which lie in lds.
template <bool ENT, bool NEAR = false> __device__ __forceinline__ Acc acc_waves(const Acc* lds, float c2) {
    const int w = threadIdx.x & 15;
    Acc a = acc_empty();
    if (w * 64 < (int)blockDim.x) a = lds[w];
    acc_rebase<ENT, NEAR>(a, lane_value(row_max(a.m), 0), c2);
    a.s = lane_value(row_sum(a.s), 0);
    if (ENT) a.e = lane_value(row_sum(a.e), 0);
    a.n = lane_value(row_sum(a.n), 0);
    return a;
}

// ------------------------------------------------------------------------------------------ who works on a row
// A workgroup, or (WAVE) each of its four waves one row: rows of a few KB, for which a barrier would cost more than it
// brings.
struct Part {
    int tid, nt, first;       // thread, threads, the wave's first thread (a scalar)
};
template <bool WAVE> __device__ __forceinline__ Part part_of() {
    if (WAVE) return {(int)(threadIdx.x & 63), 64, 0};
    return {(int)threadIdx.x, (int)blockDim.x, __builtin_amdgcn_readfirstlane(threadIdx.x) & ~63};
}
// A row cut at the 16-byte boundaries of its logits: rows of an odd vocabulary begin anywhere, and reading them in
// 16-byte steps from there was measured at 4.9 TB/s against 6.1 for aligned steps.  The logits before the first and
// behind the last boundary, up to 7 at either end, are the edge: one scalar of threads 0-6 and 8-14.
#define SHIFT_FROM 8192
template <typename T> struct Span {
    int V, head, nvec;
    int shift;                // threads before the one that takes the first vector

    __device__ __forceinline__ Span(const T* x, int V) : V(V), shift(0) {
        head = min(V, (int)(-(uintptr_t)x % 16u / sizeof(T)));
        nvec = (V - head) / VEC<T>;
    }
    // For a row whose gradient goes to `out`: the first threads stay idle so that a wave's 1 KB begins at a 128-byte line
    // of the gradient (copying rows of 50001 bf16: 5.8 TB/s against 5.3; rows of 8 KB gain nothing).
    __device__ __forceinline__ Span(const T* x, int V, const T* out) : Span(x, V) {
        if (V >= SHIFT_FROM) shift = (int)((uintptr_t)(out + head) / 16u % 8u);
    }
    __device__ __forceinline__ int edge(int tid) const {      // this thread's logit of the edge, or -1
        const int behind = head + nvec * VEC<T> + tid - 8;
        return tid < 8 ? (tid < head ? tid : -1) : (tid < 16 && behind < V ? behind : -1);
    }
};

// Vector j of the body.  KEEP: it will be read again, and a non-temporal load would let the caches drop it.
template <bool KEEP, typename T> __device__ __forceinline__ u32x4 load_vec(const T* body, int j) {
    const u32x4* at = (const u32x4*)((const char*)body + 16u * (uint32_t)j);
    return KEEP ? *at : __builtin_nontemporal_load(at);
}
// Of the gradient, whose vectors may lie across a boundary.  past: not through the caches.
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
template <typename T> __device__ __forceinline__ void store_vec(T* body, int j, u32x4 o, bool past) {
    u32x4_any* at = (u32x4_any*)((char*)body + 16u * (uint32_t)j);
    if (past) {
        asm volatile("");     // or the compiler makes one ordinary store of the two
        __builtin_nontemporal_store(o, at);
        asm volatile("");
    } else {
        *at = o;
    }
}

// (m, S, E) of `nvec` vectors and a thread's logit of the edge (-inf: none), which are not kept, joined over the wave.
// DEPTH vectors of a thread are on their way while the DEPTH before are added.
template <typename T, int DEPTH, bool ENT, bool NEAR, bool KEEP>
__device__ __forceinline__ Acc stream_stats(const T* body, int nvec, float edge, float c2, const Part& p, float counted) {
    constexpr int N = VEC<T>, M = DEPTH < 4 ? DEPTH : 4;
    Acc a = acc_empty();
    a.n = counted;
    if (nvec > 0) {
        const int step = DEPTH * p.nt, steps = nvec / step, left = nvec - steps * step;
        u32x4 v[DEPTH], next[DEPTH];
        const T* from = body;
        auto fetch = [&]() {          // a step of which every thread has its part
#pragma unroll
            for (int k = 0; k < DEPTH; ++k) next[k] = load_vec<KEEP>(from + (int64_t)k * p.nt * N, p.tid);
        };
        if (steps > 0) fetch();
        for (int i = 1; i < steps; ++i) {
            from += (int64_t)step * N;
#pragma unroll
            for (int k = 0; k < DEPTH; ++k) v[k] = next[k];
            fetch();
            __builtin_amdgcn_sched_barrier(0);    // the loads stay ahead of the arithmetic
#pragma unroll
            for (int k = 0; k < DEPTH; k += M) {
                acc_vecs<T, M, ENT, NEAR>(a, v + k, c2);
                if (DEPTH > M) __builtin_amdgcn_sched_barrier(0);    // two groups unpacked at once would not fit the registers
            }
        }
        if (steps > 0) {
#pragma unroll
            for (int k = 0; k < DEPTH; ++k) v[k] = next[k];
        }
        // the last step, which may be empty: threads without a part read the last vector of the row
#pragma unroll
        for (int k = 0; k < DEPTH; ++k) next[k] = load_vec<KEEP>(body, min(steps * step + k * p.nt + p.tid, nvec - 1));
        __builtin_amdgcn_sched_barrier(0);
        if (steps > 0) {
#pragma unroll
            for (int k = 0; k < DEPTH; k += M) {
                acc_vecs<T, M, ENT, NEAR>(a, v + k, c2);
                if (DEPTH > M) __builtin_amdgcn_sched_barrier(0);    // two groups unpacked at once would not fit the registers
            }
        }
#pragma unroll
        for (int k = 0; k < DEPTH; ++k)
            if (k * p.nt + p.first < left) {      // some lane of this wave has a part
                if (k * p.nt + p.tid >= left) next[k] = Word<T>::LOWEST;
                acc_vecs<T, 1, ENT, NEAR>(a, next + k, c2);
            }
    }
    acc_rebase<ENT, NEAR>(a, fmaxf(a.m, edge), c2);
    acc_add<ENT, NEAR>(a, edge, c2);
    return acc_wave<ENT, NEAR>(a, c2);
}

// How a forward-only kernel reads its rows: a wave each; a workgroup each; a workgroup each where there are so few rows
// that one's latency is what counts, with 8 vectors of a thread on their way (a row of 256 KB bf16: 12 us -> 10.8).
#define MODE_WAVE 0
#define MODE_BLOCK 1
#define MODE_FEW 2

// Part `seg` of `segs` of a row, joined over the workgroup in its first wave: true there, and the other waves are done.
template <typename T, int MODE, bool ENT, bool KEEP>
__device__ __forceinline__ bool stream_row(const T* x, int V, float c2, float counted, Acc* lds, Acc& a, int seg = 0,
                                           int segs = 1) {
    constexpr bool WAVE = MODE == MODE_WAVE;
    const Part p = part_of<WAVE>();
    const Span<T> s(x, V);
    const int per = (s.nvec + segs - 1) / segs, begin = min(s.nvec, seg * per), nvec = min(per, s.nvec - begin);
    const T* body = x + s.head + (int64_t)begin * VEC<T>;
    const int e = seg == 0 ? s.edge(p.tid) : -1;
    const float edge = e >= 0 ? wide(x[e]) : -__builtin_inff();
    a = stream_stats<T, MODE == MODE_FEW ? 8 : 4, ENT, true, KEEP>(body, nvec, edge, c2, p, counted);
    if (!WAVE) {
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
        __syncthreads();
        if (threadIdx.x >= 64) return false;
        a = acc_waves<ENT, true>(lds, c2);
    }
    // A row or piece that is not near is done over by this wave alone, the others being gone: 500 rows of 256 KB take 233 us
    // then and 27 otherwise.  (Nothing but -inf is not near, too.)
    const float n = a.n;
    if (is_near(a.m, c2)) a = near_done(a, c2);
    else a = stream_stats<T, 1, ENT, false, true>(body, nvec, edge, c2, part_of<true>(), 0.0f);   // the edge is the first wave's
    a.n = n;
    return true;
}

// ------------------------------------------------------------------------------------------ a row on the chip
// A row's threads hold CH vectors each, so that statistics and gradient read memory once: 16 vectors a thread are 64
// registers, and 1024 threads then hold 256 KB.  Vectors beyond are read again for the gradient.  Vector j
// belongs to thread (j + shift) % nt; lanes beside the row hold its first or last vector, not counted and not stored.
template <typename T, int CH> struct Row {
    u32x4 v[CH];
    float edge;
};

template <typename T, int CH>
__device__ __forceinline__ void row_load(Row<T, CH>& row, const T* x, const Span<T>& s, const Part& p) {
    const int e = s.edge(p.tid);
    row.edge = e >= 0 ? wide(x[e]) : -__builtin_inff();
    if (s.nvec > 0) {
#pragma unroll
        for (int i = 0; i < CH; ++i)
            row.v[i] = load_vec<false>(x + s.head, max(0, min(i * p.nt + p.tid - s.shift, s.nvec - 1)));
    }
}

// A thread's part of (m, S, E), joined over the wave, in the NEAR form.
template <typename T, int CH, bool WAVE, bool ENT>
__device__ __forceinline__ Acc row_stats(Row<T, CH>& row, const T* x, const Span<T>& s, const Part& p, float c2, float counted) {
    constexpr int M = sizeof(T) == 4 ? 4 : 2;             // vectors added at once
    const int mine = s.nvec + s.shift - p.first, tid = p.tid - s.shift;
    Acc a = acc_empty();
    a.n = counted;
#pragma unroll
    for (int i = 0; i < CH; i += M) {
        if (i * p.nt < mine) {
#pragma unroll
            for (int k = i; k < i + M; ++k)
                if ((k * p.nt + 64 > mine && k * p.nt + tid >= s.nvec) || (k == 0 && tid < 0)) row.v[k] = Word<T>::LOWEST;
            acc_vecs<T, M, ENT, true>(a, row.v + i, c2);
        }
    }
    for (int j = CH * p.nt + tid; !WAVE && j < s.nvec; j += p.nt) {
        const u32x4 v = load_vec<true>(x + s.head, j);
        acc_vecs<T, 1, ENT, true>(a, &v, c2);
    }
    acc_rebase<ENT, true>(a, fmaxf(a.m, row.edge), c2);
    acc_add<ENT, true>(a, row.edge, c2);
    return acc_wave<ENT, true>(a, c2);
}

// The exact statistics of a row that is not near, by all of its threads and in all of them.
template <typename T, bool WAVE, bool ENT>
__device__ __forceinline__ Acc far_stats(const T* x, const Span<T>& s, const Part& p, float c2, Acc* lds) {
    const int e = s.edge(p.tid);
    Acc a = stream_stats<T, 1, ENT, false, true>(x + s.head, s.nvec, e >= 0 ? wide(x[e]) : -__builtin_inff(), c2, p, 0.0f);
    if (WAVE) return a;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
    __syncthreads();
    return acc_waves<ENT>(lds, c2);
}

// ------------------------------------------------------------------------------------------ row gradient
// dL/dx_i = e_i (a + b u_i), + gt at `tok`; u_i = fma(x_i, c2, -m) in the NEAR form, (x_i - m) c2 in the other
struct RowGrad {
    float m, a, b, gt;
    int tok;     // -1: none
};

template <bool ENT, bool NEAR> __device__ __forceinline__ float grad_of(const RowGrad& g, float x, float c2) {
    const float u = NEAR ? fmaf(x, c2, -g.m) : (x - g.m) * c2;
    const float e = __builtin_amdgcn_exp2f(u);
    return ENT ? e * fmaf(g.b, fmaxf(u, U_FLOOR), g.a) : e * g.a;
}

template <typename T, bool ENT, bool NEAR>
__device__ __forceinline__ u32x4 grad_vec(const RowGrad& g, u32x4 v, int place, float c2) {   // place: of the token in v
    constexpr int N = VEC<T>;
    float d[N];
    unpack<T>(v, d);
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = grad_of<ENT, NEAR>(g, d[i], c2);
    if (place >= 0 && place < N) {
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] += i == place ? g.gt : 0.0f;
    }
    return pack<T>(d);        // the one rounding of the gradient
}

template <typename T, bool ENT, bool NEAR>
__device__ __forceinline__ void edge_grad(const RowGrad& g, float x, T* out, int i, float c2) {
    if (i < 0) return;
    const float d = grad_of<ENT, NEAR>(g, x, c2);
    out[i] = (T)(i == g.tok ? d + g.gt : d);
}

// The gradient of a held row that is near.  The vectors that are read again may lie where their gradient goes.
template <typename T, int CH, bool WAVE, bool ENT>
__device__ __forceinline__ void row_grad(const Row<T, CH>& row, const T* x, T* out, const Span<T>& s, const Part& p,
                                         float c2, const RowGrad& g, bool past) {
    constexpr int N = VEC<T>;
    const int mine = s.nvec + s.shift - p.first, tid = p.tid - s.shift;
    const int tok = g.tok >= 0 ? g.tok - s.head : -1;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        if (i * p.nt < mine) {
            const int j = i * p.nt + tid;
            const u32x4 o = grad_vec<T, ENT, true>(g, row.v[i], tok - j * N, c2);
            if (j < s.nvec && (i > 0 || j >= 0)) store_vec(out + s.head, j, o, past);
        }
    }
    for (int j = CH * p.nt + tid; !WAVE && j < s.nvec; j += p.nt)
        store_vec(out + s.head, j, grad_vec<T, ENT, true>(g, load_vec<false>(x + s.head, j), tok - j * N, c2), past);
    edge_grad<T, ENT, true>(g, row.edge, out, s.edge(p.tid), c2);
}

// Vectors, and threads before them, of a piece: whole lines of the gradient.
template <typename T> __device__ __forceinline__ int piece_of(const Span<T>& s, int segs) {
    return ((s.nvec + s.shift + segs - 1) / segs + 7) & ~7;
}

// The gradient of a row whose statistics are known, part `seg` of `segs`; x may be out.
template <typename T, bool ENT>
__device__ __forceinline__ void row_map(const T* x, T* out, int V, const Part& p, int seg, int segs, float c2,
                                        const RowGrad& g, bool past) {
    constexpr int N = VEC<T>;
    const Span<T> s(x, V, out);
    const int per = piece_of(s, segs), end = min(s.nvec, (seg + 1) * per - s.shift);
    const int tok = g.tok >= 0 ? g.tok - s.head : -1;
    int j = seg * per + p.tid - s.shift;
    if (j < 0) j += p.nt;
    for (; j < end; j += p.nt)
        store_vec(out + s.head, j, grad_vec<T, ENT, false>(g, load_vec<false>(x + s.head, j), tok - j * N, c2), past);
    const int e = seg == 0 ? s.edge(p.tid) : -1;
    edge_grad<T, ENT, false>(g, e >= 0 ? wide(x[e]) : 0.0f, out, e, c2);
}

template <typename T> __device__ __forceinline__ void row_fill(T* out, int V, const Part& p, int seg, int segs, bool past) {
    const Span<T> s(out, V, out);
    const int per = piece_of(s, segs), end = min(s.nvec, (seg + 1) * per - s.shift);
    const u32x4 zero = 0;
    int j = seg * per + p.tid - s.shift;
    if (j < 0) j += p.nt;
    for (; j < end; j += p.nt) store_vec(out + s.head, j, zero, past);
    const int e = seg == 0 ? s.edge(p.tid) : -1;
    if (e >= 0) out[e] = (T)0.0f;
}

// ------------------------------------------------------------------------------------------ launch arguments
struct Logits {
    const void* x;
    void* grad;               // may be x itself
    int64_t xs, xt, gs, gt;   // strides (elements) of sequences and tokens
    int64_t n_tok, n;         // n = sequences * n_tok rows
    int64_t r0;               // first row of this launch
    int V;
    float c, c2;              // 1/temperature; the same times log2(e)
    double ln2;               // 1/temperature / c2
    bool past;                // the gradient is stored past the caches
};

template <bool WAVE> __device__ __forceinline__ int64_t row_of(const Logits& L) {   // (one workgroup may have 16 waves)
    return L.r0 + (WAVE ? (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : (int64_t)blockIdx.x);
}

struct Place {
    uint32_t b, t;            // sequence and position
};
__device__ __forceinline__ Place place_of(const Logits& L, int64_t r) {   // rows are fewer than 2^31: one 32-bit division
    const uint32_t b = (uint32_t)r / (uint32_t)L.n_tok;
    return {b, (uint32_t)r - b * (uint32_t)L.n_tok};
}

template <typename T> __device__ __forceinline__ const T* row_in(const Logits& L, const Place& at) {
    return (const T*)L.x + (int64_t)at.b * L.xs + (int64_t)at.t * L.xt;
}
template <typename T> __device__ __forceinline__ T* row_out(const Logits& L, const Place& at) {
    return (T*)L.grad + (int64_t)at.b * L.gs + (int64_t)at.t * L.gt;
}

struct Weights {              // how much a row counts
    const uint8_t* mask;      // NULL: every row counts
    const int* seq_len;       // counted rows of each sequence
    const int* totals;        // {counted rows, sequences with one}
    int reduction;
    int count_here;           // each row's threads count the whole mask themselves
    float scale;
    int64_t n_seq;
};

#define COUNT_HERE 4096       // rows up to which that is cheaper than a launch (16 bytes of the mask are one load)
#define COUNT_SEQS 64         // and, for means over sequences, as many as a wave has lanes

// How many of 16 bytes, the first `skip` left out, are not 0.
__device__ __forceinline__ int count_16(const uint8_t* at, int skip) {
    u32x4 v;
    __builtin_memcpy(&v, at, 16);
    int k = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int out = min(max(skip - 4 * i, 0), 4) * 8;
        k += __popc((((v[i] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | v[i]) & (uint32_t)(0x80808080ull << out));
    }
    return k;
}

// This thread's part of the counted rows; for means over sequences, of 128 times those of sequence b and of the
// sequences that have one: g lanes of a wave take a sequence.
__device__ __forceinline__ float count_mask(const Weights& w, int64_t n, int64_t n_tok, uint32_t b, const Part& p) {
    int k = 0;
    if (w.count_here && w.reduction == RED_TOKEN) {
        const int whole = (int)n / 16;
        for (int j = p.tid; j < whole; j += p.nt) k += count_16(w.mask + 16 * j, 0);
        const int j = whole * 16 + p.tid;
        if (p.tid < 16 && j < (int)n) k += w.mask[j] != 0;
    } else if (w.count_here) {
        int sh = 6;
        while (((int)w.n_seq << sh) > p.nt) --sh;
        const int g = 1 << sh, mine = p.tid >> sh, lane = p.tid & (g - 1), t = (int)n_tok;
        if (p.first < ((int)w.n_seq << sh)) {     // some lane of this wave has a part
            const uint8_t* mask = w.mask + (mine < (int)w.n_seq ? mine : 0) * t;
            if (t < 16) {
                for (int c = lane; c < t; c += g) k += mask[c] != 0;
            } else {          // the last 16 bytes overlap the ones before
                for (int c = lane * 16; c < t; c += g * 16) k += count_16(mask + min(c, t - 16), max(c + 16 - t, 0));
            }
            if (mine >= (int)w.n_seq) k = 0;
            const uint64_t lanes = (g == 64 ? ~0ull : (1ull << g) - 1) << (threadIdx.x & 63 & ~(g - 1));
            const bool some = __ballot(k > 0) & lanes;
            k = (mine == (int)b ? 128 * k : 0) + (some && lane == 0);
        }
    }
    return (float)k;          // below 2^24 in any sum: exact
}

__device__ __forceinline__ float row_weight(const Weights& w, const Place& at, int64_t n_tok, float counted) {
    float d = 1.0f;           // rows are fewer than 2^30: rounded once by 2^-24 at most, as the quotient is
    if (w.reduction != RED_SUM && !w.mask) d = (float)(w.n_seq * n_tok);
    else if (w.reduction == RED_TOKEN) d = w.count_here ? counted : (float)w.totals[0];
    else if (w.reduction == RED_SEQ)
        d = w.count_here ? (float)(((int)counted >> 7) * ((int)counted & 127))
                         : (float)((int64_t)w.seq_len[at.b] * (int64_t)w.totals[1]);
    return w.scale / d;
}

struct RowStats {             // what the backward pass needs of the forward pass
    float m, s, h, w;
};

// ln S in fp64: S = 2^k f, f in [1/sqrt 2, sqrt 2), ln f = 2 artanh((f - 1) / (f + 1)) by its series (|argument| < 0.172:
// the first term left out is below 2e-11)
__device__ __forceinline__ double ln_of(float s) {
    int k;
    float f = frexpf(s, &k);
    if (!(s > 0.0f) || isinf(s)) return (double)logf(s);
    if (f < 0.70710678f) {
        f *= 2.0f;
        k -= 1;
    }
    const double den = (double)f + 1.0, guess = __builtin_amdgcn_rcp(den);     // one Newton step: beyond 2^-45
    const double z = ((double)f - 1.0) * guess * fma(-den, guess, 2.0), y = z * z;
    const double p = fma(y, fma(y, fma(y, fma(y, fma(y, 1.0 / 11, 1.0 / 9), 1.0 / 7), 1.0 / 5), 1.0 / 3), 1.0);
    return fma((double)k, LN2_D, 2.0 * z * p);
}

// The token's logit, NaN for a token that is not in the vocabulary.
template <typename T> __device__ __forceinline__ float token_logit(const T* x, int64_t tok, int V) {
    return tok >= 0 && tok < V ? wide(x[tok]) : __builtin_nanf("");
}
// ln S and ln p of a logit.  c2 is rounded: relative to 1/temperature all u_i are too long by the same factor, which
// L.ln2 takes back from a single u, and, to first order, E / S from ln S.
template <bool ENT> __device__ __forceinline__ double ln_sum(const Logits& L, const Acc& a) {
    const double ln_s = ln_of(a.s);
    return ENT ? fma(L.ln2 - LN2_D, (double)(a.e / a.s), ln_s) : ln_s;
}
template <bool NEAR> __device__ __forceinline__ double logp_of(const Logits& L, float x, float m, double ln_s) {
    const double u = NEAR ? fma((double)x, (double)L.c2, -(double)near_max(m, L.c2)) : ((double)x - (double)m) * (double)L.c2;
    const double lp = fma(L.ln2, u, -ln_s);
    return lp > 0.0 ? 0.0 : lp;        // S is rounded: no probability is above 1 for that, and no entropy below 0
}
__device__ __forceinline__ float entropy_of(const Logits& L, const Acc& a, double ln_s) {
    const float h = (float)fma(-L.ln2, (double)(a.e / a.s), ln_s);
    return h < 0.0f ? 0.0f : h;
}

// ------------------------------------------------------------------------------------------ counting masks
// One wave a sequence.  One workgroup counts everything where the mask is small; beyond, one launch counts the
// sequences and a second one (seqs_done) sums them.
__global__ __launch_bounds__(1024) void count_kernel(const uint8_t* __restrict__ mask, int64_t n_seq, int64_t n_tok,
                                                     int* seq_len, int* totals, int lens, int sums) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lens) {
        for (int64_t b = (int64_t)blockIdx.x * 16 + wave; b < n_seq; b += (int64_t)gridDim.x * 16) {
            int k = 0;
            for (int64_t t = lane; t < n_tok; t += 64) k += mask[b * n_tok + t] != 0;
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) k += __shfl_xor(k, off);
            if (lane == 0) seq_len[b] = k;
        }
    }
    if (!sums) return;
    __shared__ int part[32];
    __syncthreads();          // this workgroup's seq_len entries (all of them where lens and sums are one launch)
    int tokens = 0, seqs = 0;
    for (int64_t b = threadIdx.x; b < n_seq; b += 1024) {
        const int k = seq_len[b];
        tokens += k;
        seqs += k > 0;
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        tokens += __shfl_xor(tokens, off);
        seqs += __shfl_xor(seqs, off);
    }
    if (lane == 0) {
        part[wave] = tokens;
        part[16 + wave] = seqs;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        int k = 0;
        for (int w = 0; w < 16; ++w) k += part[16 * threadIdx.x + w];
        totals[threadIdx.x] = k;
    }
}

// The rows' losses summed in a fixed order.  One workgroup, or (loss == NULL) one of several that leave their sums for
// a second launch.
__global__ __launch_bounds__(1024) void total_kernel(const double* __restrict__ part, int64_t n, double* sums, float* loss) {
    __shared__ double lds[16];
    double s = 0.0;
    for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 1024) s += part[i];
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) s += lds[w];
        if (loss) *loss = (float)s;
        else sums[blockIdx.x] = s;
    }
}

// ------------------------------------------------------------------------------------------ log-probabilities
template <typename T, int MODE, bool ENT, bool KEEP>
__global__ __launch_bounds__(1024, 4) void logprobs_kernel(Logits L, const void* tokens, int i64, const uint8_t* mask,
                                                           float* logprobs, double* logprobs64, float* entropy,
                                                           RowStats* stats) {
    constexpr bool WAVE = MODE == MODE_WAVE;
    __shared__ Acc lds[16];
    const int64_t r = row_of<WAVE>(L);
    if (WAVE && r >= L.n) return;
    double lp = 0.0;
    RowStats st = {0.0f, 1.0f, 0.0f, 0.0f};
    if (!mask || mask[r]) {
        const T* x = row_in<T>(L, place_of(L, r));
        const float xt = token_logit(x, int_at(tokens, i64, r), L.V);
        Acc a;
        if (!stream_row<T, MODE, ENT, KEEP>(x, L.V, L.c2, 0.0f, lds, a)) return;
        const double ln_s = ln_sum<ENT>(L, a);
        lp = logp_of<false>(L, xt, a.m, ln_s);
        st.m = a.m;
        st.s = a.s;
        if (ENT) st.h = entropy_of(L, a, ln_s);
    }
    if (part_of<WAVE>().tid == 0) {
        if (logprobs) logprobs[r] = (float)lp;
        if (logprobs64) logprobs64[r] = lp;
        if (ENT && entropy) entropy[r] = st.h;
        if (stats) stats[r] = st;
    }
}

// h, ln_s: of a form's statistics; used with an entropy gradient only
__device__ __forceinline__ RowGrad grad_seed(const Logits& L, float m, float s, float h, float ln_s, float g_lp, float g_h,
                                             int64_t tok) {
    RowGrad g;
    g.m = m;
    const bool bad = tok < 0 || tok >= L.V;
    const float k = -L.c / s;
    g.a = bad ? __builtin_nanf("") : k * fmaf(g_h, h - ln_s, g_lp);
    g.b = k * g_h * (float)L.ln2;
    g.gt = L.c * g_lp;
    g.tok = bad ? -1 : (int)tok;
    return g;
}

struct Incoming {             // dL/dlogp and dL/dH of each row, and a factor on both
    const float *lp, *h, *factor;
    int64_t lp_s, lp_t, h_s, h_t;
};

// Rows in the reverse of the forward pass's order: what it read last is still in the 256 MB cache in front of the HBM.
template <typename T, bool WAVE, bool ENT>
__global__ __launch_bounds__(1024) void backward_kernel(Logits L, const void* tokens, int i64, const uint8_t* mask,
                                                       const RowStats* __restrict__ stats, Incoming in) {
    const int64_t r = L.n - 1 - row_of<WAVE>(L);
    if (WAVE && r < 0) return;
    const Part p = part_of<WAVE>();
    const Place at = place_of(L, r);
    T* out = row_out<T>(L, at);
    if (mask && !mask[r]) {
        row_fill(out, L.V, p, blockIdx.y, gridDim.y, L.past);
        return;
    }
    const float f = in.factor ? *in.factor : 1.0f;
    const RowStats st = stats[r];
    const float g_lp = in.lp ? f * in.lp[at.b * in.lp_s + at.t * in.lp_t] : 0.0f;
    const float g_h = ENT ? f * in.h[at.b * in.h_s + at.t * in.h_t] : 0.0f;
    const RowGrad g = grad_seed(L, st.m, st.s, st.h, ENT ? (float)ln_of(st.s) : 0.0f, g_lp, g_h, int_at(tokens, i64, r));
    row_map<T, ENT>(row_in<T>(L, at), out, L.V, p, blockIdx.y, gridDim.y, L.c2, g, L.past);
}

// ------------------------------------------------------------------------------------------ clipped policy loss
struct PolicyArgs {
    const void* tokens;
    int i64;
    const float *old_lp, *adv, *ref;
    int64_t adv_s, adv_t;
    float lo, hi, kl, ent;    // clip range of the ratio, coefficients
    Weights w;
    float *logprobs, *entropy;
    RowStats* stats;          // with seeds: the differentiable form
    float *g_lp, *g_h;
    double* part;             // weighted loss of each row
    float* solo;              // the loss, where one workgroup has all rows
};

// Gradients of a counted row's loss, and the parts that the loss itself is made of afterwards.
struct PolicyRow {
    float g_lp, g_h, w, kl;
    double surrogate;
};

__device__ __forceinline__ PolicyRow policy_row(const PolicyArgs& p, double lp, float old_lp, float adv, float ref, float w) {
    // Differences of log-probabilities are formed in fp64, where they lose nothing.  The ratio is 1 + (e^d - 1) with
    // the second part in fp32: near 1 that keeps more of it than fp32 does, and a loss is a mean in which A and -A
    // nearly cancel.
    PolicyRow o;
    const double r = 1.0 + (double)expm1f((float)(lp - (double)old_lp)), a = (double)adv;
    const bool clipped = (adv > 0.0f && r > (double)p.hi) || (adv < 0.0f && r < (double)p.lo);
    o.surrogate = clipped ? (adv > 0.0f ? (double)p.hi : (double)p.lo) * a : r * a;
    float g = clipped ? 0.0f : (float)(-r * a);
    o.kl = 0.0f;
    if (p.kl != 0.0f) {
        const float d = (float)((double)ref - lp);
        // e^d - 1 - d: its series where the difference would cancel (|d|^6 / 20160 < 2^-24 at 1/4)
        const float em1 = expm1f(d);
        o.kl = fabsf(d) < 0.25f
            ? d * d * fmaf(d, fmaf(d, fmaf(d, fmaf(d, fmaf(d, 1.0f / 5040, 1.0f / 720), 1.0f / 120), 1.0f / 24), 1.0f / 6), 0.5f)
            : em1 - fminf(d, __FLT_MAX__);     // an impossible token: infinite, not the difference of two infinities
        g = fmaf(-p.kl, em1, g);
    }
    o.g_lp = w * g;
    o.g_h = -w * p.ent;
    o.w = w;
    return o;
}

__device__ __forceinline__ double weighted_loss(const PolicyArgs& p, const PolicyRow& o, float h) {
    double loss = -o.surrogate;
    if (p.kl != 0.0f) loss = fma((double)p.kl, (double)o.kl, loss);
    if (p.ent != 0.0f) loss = fma(-(double)p.ent, (double)h, loss);
    return o.w != 0.0f ? loss * (double)o.w : 0.0;      // a row that does not count
}

// inputs of a counted row
struct PolicyIn {
    float xt, old_lp, adv, ref;
    int64_t tok;
};
template <typename T>
__device__ __forceinline__ PolicyIn policy_in(const Logits& L, const PolicyArgs& p, const T* x, int64_t r, const Place& at) {
    PolicyIn i;
    i.tok = int_at(p.tokens, p.i64, r);
    i.old_lp = p.old_lp[r];
    i.adv = p.adv[at.b * p.adv_s + at.t * p.adv_t];
    i.ref = p.ref ? p.ref[r] : 0.0f;
    i.xt = token_logit(x, i.tok, L.V);
    return i;
}

// The weighted loss of row r: left to total_kernel, or, where this workgroup has all rows, summed over its waves in their
// order (every wave comes here then, with 0 where it had no row).
template <bool WAVE> __device__ __forceinline__ void row_loss(const PolicyArgs& p, int64_t r, int64_t n, double loss) {
    if (!p.solo) {
        if (part_of<WAVE>().tid == 0 && r < n) p.part[r] = loss;
        return;
    }
    __shared__ double sums[16];
    if (WAVE) {
        if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = loss;
        __syncthreads();
        if (threadIdx.x == 0) {
            loss = 0.0;
            for (int w = 0; w < (int)blockDim.x / 64; ++w) loss += sums[w];
        }
    }
    if (threadIdx.x == 0) *p.solo = (float)loss;
}

// A counted row from its statistics to what the loss and its gradient need of it.
struct PolicyDone {
    double lp, ln_s;
    float h;
    PolicyRow o;
};
template <bool NEAR>
__device__ __forceinline__ PolicyDone policy_done(const Logits& L, const PolicyArgs& p, const PolicyIn& in, const Acc& a,
                                                  const Place& at, float counted) {
    PolicyDone d;
    d.ln_s = ln_sum<true>(L, a);
    d.lp = logp_of<NEAR>(L, in.xt, a.m, d.ln_s);
    d.h = entropy_of(L, a, d.ln_s);
    d.o = policy_row(p, d.lp, in.old_lp, in.adv, in.ref, row_weight(p.w, at, L.n_tok, counted));
    return d;
}
__device__ __forceinline__ RowGrad policy_seed(const Logits& L, const PolicyDone& d, float m, float s, int64_t tok) {
    return grad_seed(L, m, s, d.h, (float)d.ln_s, d.o.g_lp, d.o.g_h, tok);
}

// Forward only; leaves what the backward pass needs.
template <typename T, int MODE>
__global__ __launch_bounds__(1024, 4) void policy_forward_kernel(Logits L, PolicyArgs p) {
    constexpr bool WAVE = MODE == MODE_WAVE;
    __shared__ Acc lds[16];
    const int64_t r = row_of<WAVE>(L);
    PolicyDone d = {};
    if (!WAVE || r < L.n) {
        RowStats st = {0.0f, 1.0f, 0.0f, 0.0f};
        if (!p.w.mask || p.w.mask[r]) {
            const Place at = place_of(L, r);
            const T* x = row_in<T>(L, at);
            const PolicyIn in = policy_in(L, p, x, r, at);
            Acc a;
            if (!stream_row<T, MODE, true, true>(x, L.V, L.c2, count_mask(p.w, L.n, L.n_tok, at.b, part_of<WAVE>()), lds, a)) return;
            d = policy_done<false>(L, p, in, a, at, a.n);
            st = {a.m, a.s, d.h, 0.0f};
        }
        if (part_of<WAVE>().tid == 0) {
            p.logprobs[r] = (float)d.lp;
            if (p.entropy) p.entropy[r] = d.h;
            if (p.stats) {
                p.stats[r] = st;
                p.g_lp[r] = d.o.g_lp;
                p.g_h[r] = d.o.g_h;
            }
        }
    }
    row_loss<WAVE>(p, r, L.n, weighted_loss(p, d.o, d.h));
}

// Loss and gradient: the row stays on the chip between its statistics and its gradient.  The first wave makes of the
// statistics what all others need (a row's fp64 arithmetic is some 300 instructions, as much as 30 vectors' gradient).
struct RowShared {
    Acc acc[16];
    RowGrad grad;
    int near_;
};

template <typename T, int CH, bool WAVE, bool ENT_GRAD>
__global__ __launch_bounds__(1024, 4) void policy_kernel(Logits L, PolicyArgs p) {
    __shared__ RowShared sh;
    const Part q = part_of<WAVE>();
    const int64_t r = row_of<WAVE>(L);
    PolicyDone d = {};
    if (!WAVE || r < L.n) {
        const Place at = place_of(L, r);
        T* out = row_out<T>(L, at);
        if (!p.w.mask || p.w.mask[r]) {
            const T* x = row_in<T>(L, at);
            const Span<T> s = WAVE ? Span<T>(x, L.V) : Span<T>(x, L.V, out);
            Row<T, CH> row;
            const PolicyIn in = policy_in(L, p, x, r, at);
            row_load(row, x, s, q);
            const float counted = count_mask(p.w, L.n, L.n_tok, at.b, q);
            asm volatile("" :: "v"(in.xt));   // read before the barrier: the gradient may overwrite it
            Acc a = row_stats<T, CH, WAVE, true>(row, x, s, q, L.c2, counted);
            RowGrad g;
            bool near_ = true;
            if (!WAVE) {
                if ((threadIdx.x & 63) == 0) sh.acc[threadIdx.x >> 6] = a;
                __syncthreads();
            }
            if (WAVE || q.first == 0) {
                if (!WAVE) a = acc_waves<true, true>(sh.acc, L.c2);
                near_ = is_near(a.m, L.c2);
                d = policy_done<true>(L, p, in, a, at, a.n);
                g = policy_seed(L, d, near_max(a.m, L.c2), a.s, in.tok);
                if (!WAVE && threadIdx.x == 0) {
                    sh.grad = g;
                    sh.near_ = near_;
                }
            }
            if (!WAVE) {
                __syncthreads();
                g = sh.grad;
                near_ = sh.near_;
            }
            if (near_) {
                row_grad<T, CH, WAVE, ENT_GRAD>(row, x, out, s, q, L.c2, g, L.past);
            } else {
                const float n = a.n;
                a = far_stats<T, WAVE, true>(x, s, q, L.c2, sh.acc);
                d = policy_done<false>(L, p, in, a, at, n);      // (n: the first wave's, which alone uses the weighted results)
                if (!WAVE) {
                    if (threadIdx.x == 0) sh.grad = policy_seed(L, d, a.m, a.s, in.tok);
                    __syncthreads();
                    g = sh.grad;
                } else {
                    g = policy_seed(L, d, a.m, a.s, in.tok);
                }
                row_map<T, ENT_GRAD>(x, out, L.V, q, 0, 1, L.c2, g, L.past);
            }
        } else {
            row_fill(out, L.V, q, 0, 1, L.past);
        }
        if (q.tid == 0) {
            p.logprobs[r] = (float)d.lp;
            if (p.entropy) p.entropy[r] = d.h;
        }
    }
    row_loss<WAVE>(p, r, L.n, weighted_loss(p, d.o, d.h));
}

// Rows of at most 256 logits: G lanes a row, at most 16 logits a lane (8 of a lane that has a row, as of a head of a few
// actions, by itself), element by element.  A wave's fp64 arithmetic then serves 64 / G rows: 524288 rows of 6 logits
// with their gradient take 21 us with a lane each, 36 with four and took 413 with a wave.
template <typename T, int G> struct Tiny {
    static constexpr int PER = G == 1 ? 8 : 16;
    float f[PER];
    int lane;

    __device__ __forceinline__ Acc load(const T* x, int V, float c2) {
        lane = threadIdx.x & (G - 1);
        Acc a = acc_empty();
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            f[k] = -__builtin_inff();
            if (k * G + lane < V) f[k] = wide(x[k * G + lane]);
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) a.m = fmaxf(a.m, f[k]);
        a.m = group(a.m, [](float p, float q) { return fmaxf(p, q); });
#pragma unroll
        for (int k = 0; k < PER; ++k)
            if (k * G < V) acc_add<true>(a, f[k], c2);
        a.s = group(a.s, [](float p, float q) { return p + q; });
        a.e = group(a.e, [](float p, float q) { return p + q; });
        return a;
    }
    // over the G lanes of a row, the same bits in each
    template <typename F> static __device__ __forceinline__ float group(float v, F op) {
        if (G == 16) {
            v = op(v, ror<0x128>(v));
            v = op(v, ror<0x124>(v));
        }
        if (G == 1) return v;
        v = op(v, ror<0x4e>(v));   // quads: lanes 2, 3, 0, 1
        return op(v, ror<0xb1>(v));   // lanes 1, 0, 3, 2
    }
    __device__ __forceinline__ void store(T* out, int V, float c2, const RowGrad& g) const {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int i = k * G + lane;
            if (i < V) {
                const float d = grad_of<true, false>(g, f[k], c2);
                out[i] = (T)(i == g.tok ? d + g.gt : d);
            }
        }
    }
    static __device__ __forceinline__ void zero(T* out, int V) {
        for (int i = threadIdx.x & (G - 1); i < V; i += G) out[i] = (T)0.0f;
    }
    static __device__ __forceinline__ int64_t row(const Logits& L) {
        return L.r0 + ((int64_t)blockIdx.x * 256 + threadIdx.x) / G;
    }
};

template <typename T, int G>
__global__ __launch_bounds__(256) void tiny_logprobs_kernel(Logits L, const void* tokens, int i64, const uint8_t* mask,
                                                            float* logprobs, double* logprobs64, float* entropy, RowStats* stats) {
    const int64_t r = Tiny<T, G>::row(L);
    if (r >= L.n) return;
    double lp = 0.0;
    RowStats st = {0.0f, 1.0f, 0.0f, 0.0f};
    if (!mask || mask[r]) {
        const T* x = row_in<T>(L, place_of(L, r));
        Tiny<T, G> row;
        const Acc a = row.load(x, L.V, L.c2);
        const double ln_s = ln_sum<true>(L, a);
        lp = logp_of<false>(L, token_logit(x, int_at(tokens, i64, r), L.V), a.m, ln_s);
        st = {a.m, a.s, entropy_of(L, a, ln_s), 0.0f};
    }
    if (threadIdx.x & (G - 1)) return;
    if (logprobs) logprobs[r] = (float)lp;
    if (logprobs64) logprobs64[r] = lp;
    if (entropy) entropy[r] = st.h;
    if (stats) stats[r] = st;
}

template <typename T, int G>
__global__ __launch_bounds__(256) void tiny_backward_kernel(Logits L, const void* tokens, int i64, const uint8_t* mask,
                                                            const RowStats* __restrict__ stats, Incoming in) {
    const int64_t r = Tiny<T, G>::row(L);
    if (r >= L.n) return;
    const Place at = place_of(L, r);
    if (mask && !mask[r]) {
        Tiny<T, G>::zero(row_out<T>(L, at), L.V);
        return;
    }
    Tiny<T, G> row;
    row.load(row_in<T>(L, at), L.V, L.c2);
    const float f = in.factor ? *in.factor : 1.0f;
    const RowStats st = stats[r];
    const float g_lp = in.lp ? f * in.lp[at.b * in.lp_s + at.t * in.lp_t] : 0.0f;
    const float g_h = in.h ? f * in.h[at.b * in.h_s + at.t * in.h_t] : 0.0f;
    row.store(row_out<T>(L, at), L.V, L.c2,
              grad_seed(L, st.m, st.s, st.h, in.h ? (float)ln_of(st.s) : 0.0f, g_lp, g_h, int_at(tokens, i64, r)));
}

// Loss, and the gradient (GRAD) or what a backward pass needs.
template <typename T, int G, bool GRAD>
__global__ __launch_bounds__(256) void tiny_policy_kernel(Logits L, PolicyArgs p) {
    const int64_t r = Tiny<T, G>::row(L);
    if (r >= L.n) return;
    const Place at = place_of(L, r);
    PolicyDone d = {};
    RowStats st = {0.0f, 1.0f, 0.0f, 0.0f};
    if (!p.w.mask || p.w.mask[r]) {
        const T* x = row_in<T>(L, at);
        const PolicyIn in = policy_in(L, p, x, r, at);
        Tiny<T, G> row;
        const Acc a = row.load(x, L.V, L.c2);
        d = policy_done<false>(L, p, in, a, at, 0.0f);
        st = {a.m, a.s, d.h, 0.0f};
        if (GRAD) row.store(row_out<T>(L, at), L.V, L.c2, policy_seed(L, d, a.m, a.s, in.tok));
    } else if (GRAD) {
        Tiny<T, G>::zero(row_out<T>(L, at), L.V);
    }
    if (threadIdx.x & (G - 1)) return;
    p.logprobs[r] = (float)d.lp;
    if (p.entropy) p.entropy[r] = d.h;
    if (!GRAD && p.stats) {
        p.stats[r] = st;
        p.g_lp[r] = d.o.g_lp;
        p.g_h[r] = d.o.g_h;
    }
    const double loss = weighted_loss(p, d.o, d.h);
    if (p.solo) *p.solo = (float)loss;     // the only row
    else p.part[r] = loss;
}

// Few long rows: a row in `parts` pieces of a workgroup each, first their statistics (split_stats_kernel), then, in a
// second launch, the row's loss and the pieces' gradients.  The first launch also takes along what of the logits the
// second needs beside its piece, which another workgroup of that launch may have overwritten.
#define SPLIT_PARTS 64
struct Split {
    Acc* acc;                 // n * parts; n of a row's first one: the token's logit
    int* teach;               // entries of each row (distillation)
    int parts;
};

// blockIdx.y: the piece
template <typename T, bool ENT>
__global__ __launch_bounds__(256) void split_stats_kernel(Logits L, const uint8_t* mask, const void* tokens, int i64, Split sp) {
    __shared__ Acc lds[16];
    const int64_t r = blockIdx.x;
    if (mask && !mask[r]) return;
    const T* x = row_in<T>(L, place_of(L, r));
    const float xt = tokens && blockIdx.y == 0 ? token_logit(x, int_at(tokens, i64, r), L.V) : 0.0f;
    Acc a;
    if (!stream_row<T, MODE_BLOCK, ENT, true>(x, L.V, L.c2, 0.0f, lds, a, blockIdx.y, sp.parts)) return;
    a.n = xt;
    if (threadIdx.x == 0) sp.acc[r * sp.parts + blockIdx.y] = a;
}

// A row's pieces joined, by a wave and in all of its lanes.
template <bool ENT> __device__ __forceinline__ Acc split_join(const Split& sp, int64_t r, float c2) {
    const int lane = threadIdx.x & 63;
    Acc a = acc_empty();
    if (lane < sp.parts) a = sp.acc[r * sp.parts + lane];
    a.n = 0.0f;
    return acc_wave<ENT>(a, c2);
}

// Log-probabilities of rows that were cut, a wave each.
template <bool ENT>
__global__ __launch_bounds__(256) void split_logprobs_kernel(Logits L, const uint8_t* mask, float* logprobs, double* logprobs64,
                                                             float* entropy, RowStats* stats, Split sp) {
    const int64_t r = row_of<true>(L);
    if (r >= L.n) return;
    double lp = 0.0;
    RowStats st = {0.0f, 1.0f, 0.0f, 0.0f};
    if (!mask || mask[r]) {
        const Acc a = split_join<ENT>(sp, r, L.c2);
        const double ln_s = ln_sum<ENT>(L, a);
        lp = logp_of<false>(L, sp.acc[r * sp.parts].n, a.m, ln_s);
        st = {a.m, a.s, ENT ? entropy_of(L, a, ln_s) : 0.0f, 0.0f};
    }
    if ((threadIdx.x & 63) > 0) return;
    if (logprobs) logprobs[r] = (float)lp;
    if (logprobs64) logprobs64[r] = lp;
    if (ENT && entropy) entropy[r] = st.h;
    if (stats) stats[r] = st;
}

template <typename T, bool ENT_GRAD>
__global__ __launch_bounds__(256) void policy_split_kernel(Logits L, PolicyArgs p, Split sp) {
    __shared__ RowShared sh;
    const Part q = part_of<false>();
    const int64_t r = blockIdx.x;
    const Place at = place_of(L, r);
    T* out = row_out<T>(L, at);
    PolicyDone d = {};
    if (!p.w.mask || p.w.mask[r]) {
        if (q.first == 0) {
            PolicyIn in;
            in.tok = int_at(p.tokens, p.i64, r);
            in.old_lp = p.old_lp[r];
            in.adv = p.adv[at.b * p.adv_s + at.t * p.adv_t];
            in.ref = p.ref ? p.ref[r] : 0.0f;
            in.xt = sp.acc[r * sp.parts].n;
            const Acc a = split_join<true>(sp, r, L.c2);
            d = policy_done<false>(L, p, in, a, at, wave_sum(count_mask(p.w, L.n, L.n_tok, at.b, part_of<true>())));
            if (threadIdx.x == 0) sh.grad = policy_seed(L, d, a.m, a.s, in.tok);
        }
        __syncthreads();
        row_map<T, ENT_GRAD>(row_in<T>(L, at), out, L.V, q, blockIdx.y, gridDim.y, L.c2, sh.grad, L.past);
    } else {
        row_fill(out, L.V, q, blockIdx.y, gridDim.y, L.past);
    }
    if (blockIdx.y > 0) return;
    if (threadIdx.x == 0) {
        p.logprobs[r] = (float)d.lp;
        if (p.entropy) p.entropy[r] = d.h;
    }
    row_loss<false>(p, r, L.n, weighted_loss(p, d.o, d.h));
}

// ------------------------------------------------------------------------------------------ preference loss
// One workgroup a pair: both sequences' sums in fp64, the pair's loss and dL/dlogp of all of a sequence's tokens.
__global__ __launch_bounds__(256) void pair_kernel(const double* __restrict__ lp, const uint8_t* __restrict__ mask,
                                                   const float* __restrict__ ref, int64_t n_pairs, int64_t n_tok,
                                                   double beta, double smooth, double scale, float* rewards,
                                                   float* seeds, double* part, float* solo) {
    __shared__ double lds[4];
    for (int64_t q = blockIdx.x; q < n_pairs; q += gridDim.x) {
        double s[2];
        for (int side = 0; side < 2; ++side) {
            const int64_t at = (q + side * n_pairs) * n_tok;
            double a = 0.0;
            for (int64_t t = threadIdx.x; t < n_tok; t += 256)
                if (!mask || mask[at + t]) a += lp[at + t];
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) a += __shfl_xor(a, off);
            __syncthreads();
            if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
            __syncthreads();
            s[side] = beta * (((lds[0] + lds[1]) + (lds[2] + lds[3])) - (double)ref[q + side * n_pairs]);
        }
        if (threadIdx.x == 0) {
            const double z = s[0] - s[1], t = exp(-fabs(z)), l = log1p(t);   // ln(1 + e^-|z|)
            const double neg = (z > 0.0 ? 0.0 : -z) + l, pos = (z > 0.0 ? z : 0.0) + l;   // -ln sig(z), -ln sig(-z); NaN stays in l
            const double sig = z > 0.0 ? 1.0 / (1.0 + t) : t / (1.0 + t);
            // both may be inf, where the other one alone may count
            const double loss = scale * ((smooth != 1.0 ? (1.0 - smooth) * neg : 0.0) + (smooth != 0.0 ? smooth * pos : 0.0)) / (double)n_pairs;
            if (solo) *solo = (float)loss;     // the only pair
            else part[q] = loss;
            const float g = (float)(scale * beta * (sig - (1.0 - smooth)) / (double)n_pairs);
            rewards[q] = (float)s[0];
            rewards[q + n_pairs] = (float)s[1];
            seeds[q] = g;
            seeds[q + n_pairs] = -g;
        }
    }
}

// ------------------------------------------------------------------------------------------ distillation
struct TeacherArgs {
    const void *index, *logit;
    int i64, dtype, K;
    Weights w;
    float* losses;
    RowStats* stats;
    const float* factor;
    double* part;
    float* solo;              // the loss, where there is one row
};

// One row's entries, K of each array in LDS.  The first wave makes them while the others wait for their logits.
struct Teacher {
    int* index;               // -1: padding
    float* q;                 // the teacher's probability of the entry
    float* x;                 // the policy's logit there
    int* bad;                 // a token beyond the vocabulary
    int* some;                // an entry that is not padding
    __device__ __forceinline__ Teacher(int* lds, int K)
        : index(lds + 2), q((float*)(lds + 2 + K)), x((float*)(lds + 2 + 2 * K)), bad(lds), some(lds + 1) {}
};
static size_t teacher_lds(int K) { return (size_t)(2 + 3 * K) * 4; }
#define TEACHER_WORDS (4 + 3 * PPO_MAX_TEACHER_TOP)      // the same of a row in memory: bad, some, sum q ln q, then the arrays

// First wave only.  Returns sum q ln q.
template <typename T>
__device__ __forceinline__ float teacher_load(const TeacherArgs& p, const Logits& L, int64_t r, const T* x, const Teacher& s) {
    const int lane = threadIdx.x;
    float mx = -__FLT_MAX__, total = 0.0f, ent = 0.0f;
    bool bad = false, some = false;
    for (int k = lane; k < p.K; k += 64) {
        const int64_t i = int_at(p.index, p.i64, r * p.K + k);
        const float t = float_at(p.logit, p.dtype, r * p.K + k);
        const bool there = i >= 0 && i < L.V;
        bad |= i >= L.V;
        some |= there;
        s.index[k] = there ? (int)i : -1;
        s.q[k] = t;
        s.x[k] = there ? wide(x[i]) : 0.0f;
        if (there) mx = fmaxf(mx, t);
    }
    mx = wave_max(mx);
    for (int k = lane; k < p.K; k += 64) total += s.index[k] >= 0 ? expf((s.q[k] - mx) * L.c) : 0.0f;
    total = wave_sum(total);
    const float lt = (float)ln_of(total);
    for (int k = lane; k < p.K; k += 64) {
        const float d = (s.q[k] - mx) * L.c, q = s.index[k] >= 0 ? expf(d) / total : 0.0f;
        s.q[k] = q;
        if (q != 0.0f) ent = fmaf(q, d - lt, ent);
    }
    bad = __any(bad);
    some = __any(some);
    if (lane == 0) {
        *s.bad = bad;
        *s.some = some;
    }
    return wave_sum(ent);
}

// First wave only: sum q (ln q - ln p).
__device__ __forceinline__ float teacher_loss(const TeacherArgs& p, const Teacher& s, float ent, const Acc& a, const Logits& L) {
    const double ln_s = ln_sum<false>(L, a);
    double cross = 0.0;
    for (int k = threadIdx.x; k < p.K; k += 64)
        if (s.q[k] != 0.0f) cross += (double)s.q[k] * logp_of<false>(L, s.x[k], a.m, ln_s);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) cross += __shfl_xor(cross, off);
    return *s.bad ? __builtin_nanf("") : (float)((double)ent - cross);
}

// dL/dx_i = g (p_i - sum of the teacher's q at i): the bulk first, the K places after a barrier.
__device__ __forceinline__ RowGrad teacher_seed(const Teacher& s, float m, float sum, float g) {
    return {m, *s.bad ? __builtin_nanf("") : g / sum, 0.0f, 0.0f, -1};
}
// A teacher that gave padding only teaches nothing: zeros, whatever the logits are (0 times a NaN is none).
__device__ __forceinline__ bool teaches(const Teacher& s) { return *s.bad || *s.some; }

template <typename T, bool NEAR>
__device__ __forceinline__ void teacher_places(const TeacherArgs& p, const Teacher& s, T* out, const Logits& L,
                                               const RowGrad& rg, float g, const Span<T>& w, int seg = 0, int segs = 1) {
    // The bulk is written, and has arrived: other waves' stores to these places come first (no cost was measured).
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (*s.bad) return;
    const int per = piece_of(w, segs);
    for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
        const int i = s.index[k];
        if (i < 0) continue;
        if (segs > 1) {       // of this piece only; the edge is the first one's
            const int j = i < w.head ? -1 : (i - w.head) / VEC<T>;
            if ((j < 0 || j >= w.nvec ? 0 : (j + w.shift) / per) != seg) continue;
        }
        float all = 0.0f;     // a token that appears twice: both entries, in both places the same number
        for (int j = 0; j < p.K; ++j) all += s.index[j] == i ? s.q[j] : 0.0f;
        out[i] = (T)(grad_of<false, NEAR>(rg, s.x[k], L.c2) - g * all);
    }
}

template <typename T, int MODE>
__global__ __launch_bounds__(1024, 4) void distill_forward_kernel(Logits L, TeacherArgs p) {
    __shared__ Acc lds[16];
    extern __shared__ int entries[];
    const Teacher teach(entries, p.K);
    const int64_t r = row_of<false>(L);
    RowStats st = {0.0f, 1.0f, 0.0f, 0.0f};
    float loss = 0.0f;
    if (!p.w.mask || p.w.mask[r]) {
        const Place at = place_of(L, r);
        const T* x = row_in<T>(L, at);
        float ent = 0.0f;
        if (threadIdx.x < 64) ent = teacher_load(p, L, r, x, teach);
        Acc a;
        if (!stream_row<T, MODE, false, true>(x, L.V, L.c2, count_mask(p.w, L.n, L.n_tok, at.b, part_of<false>()), lds, a)) return;
        loss = teacher_loss(p, teach, ent, a, L) / (L.c * L.c);
        st.m = a.m;
        st.s = a.s;
        st.w = row_weight(p.w, at, L.n_tok, a.n);
    }
    if (threadIdx.x == 0) {
        if (p.losses) p.losses[r] = loss;
        if (p.stats) p.stats[r] = st;
        if (p.solo) *p.solo = (float)((double)st.w * (double)loss);
        else p.part[r] = (double)st.w * (double)loss;
    }
}

template <typename T, int CH>
__global__ __launch_bounds__(1024, 4) void distill_kernel(Logits L, TeacherArgs p) {
    __shared__ RowShared sh;
    extern __shared__ int entries[];
    const Teacher teach(entries, p.K);
    const int64_t r = row_of<false>(L);
    const Part q = part_of<false>();
    const Place at = place_of(L, r);
    T* out = row_out<T>(L, at);
    float loss = 0.0f, w = 0.0f;
    if (!p.w.mask || p.w.mask[r]) {
        const T* x = row_in<T>(L, at);
        const Span<T> s(x, L.V, out);
        Row<T, CH> row;
        row_load(row, x, s, q);
        float ent = 0.0f;
        if (q.first == 0) ent = teacher_load(p, L, r, x, teach);
        Acc a = row_stats<T, CH, false, false>(row, x, s, q, L.c2, count_mask(p.w, L.n, L.n_tok, at.b, q));
        if ((threadIdx.x & 63) == 0) sh.acc[threadIdx.x >> 6] = a;
        __syncthreads();
        a = acc_waves<false, true>(sh.acc, L.c2);
        w = row_weight(p.w, at, L.n_tok, a.n);
        const float scale = w / L.c;
        if (!teaches(teach)) {
            row_fill(out, L.V, q, 0, 1, L.past);
        } else if (is_near(a.m, L.c2)) {
            const RowGrad g = teacher_seed(teach, near_max(a.m, L.c2), a.s, scale);
            row_grad<T, CH, false, false>(row, x, out, s, q, L.c2, g, L.past);
            teacher_places<T, true>(p, teach, out, L, g, scale, s);
            a = near_done(a, L.c2);
        } else {
            __syncthreads();  // sh.acc has been read
            a = far_stats<T, false, false>(x, s, q, L.c2, sh.acc);
            const RowGrad g = teacher_seed(teach, a.m, a.s, scale);
            row_map<T, false>(x, out, L.V, q, 0, 1, L.c2, g, L.past);
            teacher_places<T, false>(p, teach, out, L, g, scale, s);
        }
        if (q.first == 0) loss = teacher_loss(p, teach, ent, a, L) / (L.c * L.c);
    } else {
        row_fill(out, L.V, q, 0, 1, L.past);
    }
    if (threadIdx.x == 0) {
        if (p.losses) p.losses[r] = loss;
        if (p.solo) *p.solo = (float)((double)w * (double)loss);
        else p.part[r] = (double)w * (double)loss;
    }
}

// Few long rows, as policy_split_kernel.  A workgroup beside the pieces' makes the teacher's entries, because another
// piece's gradient may lie where the policy's logits of the entries were.
template <typename T> __global__ __launch_bounds__(256) void split_teacher_kernel(Logits L, TeacherArgs p, Split sp) {
    __shared__ Acc lds[16];
    extern __shared__ int entries[];
    const int64_t r = blockIdx.x;
    if (p.w.mask && !p.w.mask[r]) return;
    const T* x = row_in<T>(L, place_of(L, r));
    if ((int)blockIdx.y < sp.parts) {
        Acc a;
        if (!stream_row<T, MODE_BLOCK, false, true>(x, L.V, L.c2, 0.0f, lds, a, blockIdx.y, sp.parts)) return;
        if (threadIdx.x == 0) sp.acc[r * sp.parts + blockIdx.y] = a;
        return;
    }
    const Teacher teach(entries, p.K);
    float ent = 0.0f;
    if (threadIdx.x < 64) ent = teacher_load(p, L, r, x, teach);
    __syncthreads();
    int* to = sp.teach + r * TEACHER_WORDS;
    for (int k = threadIdx.x; k < 2 + 3 * p.K; k += 256) to[k < 2 ? k : k + 2] = entries[k];
    if (threadIdx.x == 0) to[2] = __float_as_int(ent);
}

template <typename T> __global__ __launch_bounds__(256) void distill_split_kernel(Logits L, TeacherArgs p, Split sp) {
    extern __shared__ int entries[];
    __shared__ Acc joined;
    const Teacher teach(entries, p.K);
    const int64_t r = blockIdx.x;
    const Part q = part_of<false>();
    const Place at = place_of(L, r);
    T* out = row_out<T>(L, at);
    float loss = 0.0f, w = 0.0f;
    if (!p.w.mask || p.w.mask[r]) {
        const int* from = sp.teach + r * TEACHER_WORDS;
        for (int k = threadIdx.x; k < 2 + 3 * p.K; k += 256) entries[k] = from[k < 2 ? k : k + 2];
        if (q.first == 0) {
            Acc a = split_join<false>(sp, r, L.c2);
            a.n = wave_sum(count_mask(p.w, L.n, L.n_tok, at.b, part_of<true>()));
            if (threadIdx.x == 0) joined = a;
        }
        __syncthreads();
        const Acc a = joined;
        w = row_weight(p.w, at, L.n_tok, a.n);
        const T* x = row_in<T>(L, at);
        if (teaches(teach)) {
            const RowGrad g = teacher_seed(teach, a.m, a.s, w / L.c);
            row_map<T, false>(x, out, L.V, q, blockIdx.y, gridDim.y, L.c2, g, L.past);
            teacher_places<T, false>(p, teach, out, L, g, w / L.c, Span<T>(x, L.V, out), blockIdx.y, gridDim.y);
        } else {
            row_fill(out, L.V, q, blockIdx.y, gridDim.y, L.past);
        }
        if (q.first == 0) loss = teacher_loss(p, teach, __int_as_float(from[2]), a, L) / (L.c * L.c);
    } else {
        row_fill(out, L.V, q, blockIdx.y, gridDim.y, L.past);
    }
    if (threadIdx.x > 0 || blockIdx.y > 0) return;
    if (p.losses) p.losses[r] = loss;
    if (p.solo) *p.solo = (float)((double)w * (double)loss);
    else p.part[r] = (double)w * (double)loss;
}

template <typename T> __global__ __launch_bounds__(1024) void distill_backward_kernel(Logits L, TeacherArgs p) {
    extern __shared__ int entries[];
    const Teacher teach(entries, p.K);
    const int64_t r = L.n - 1 - row_of<false>(L);   // as in backward_kernel
    const Part q = part_of<false>();
    const Place at = place_of(L, r);
    T* out = row_out<T>(L, at);
    if (p.w.mask && !p.w.mask[r]) {
        row_fill(out, L.V, q, 0, 1, L.past);
        return;
    }
    const T* x = row_in<T>(L, at);
    if (q.first == 0) teacher_load(p, L, r, x, teach);
    __syncthreads();
    if (!teaches(teach)) {
        row_fill(out, L.V, q, 0, 1, L.past);
        return;
    }
    const RowStats st = p.stats[r];
    const float g = (p.factor ? *p.factor : 1.0f) * st.w / L.c;
    const RowGrad rg = teacher_seed(teach, st.m, st.s, g);
    row_map<T, false>(x, out, L.V, q, 0, 1, L.c2, rg, L.past);
    teacher_places<T, false>(p, teach, out, L, rg, g, Span<T>(x, L.V, out));
}

// ------------------------------------------------------------------------------------------ host side
#define ALIGN256(n) (((size_t)(n) + 255) & ~(size_t)255)

#define TOTAL_GRID 64
#define SPLIT_ROWS 128        // rows that are ever cut

struct Workspace {            // one call's scratch
    double *part, *sums;      // weighted loss of each row (or pair); TOTAL_GRID sums of them
    int *totals, *seq_len;
    double* lp64;             // the pairs' log-probabilities
    float* seeds;             // and their gradients
    RowStats* stats;
    Acc* acc;                 // statistics of pieces of few long rows
    int* teach;               // and their teacher's entries
    size_t bytes;
};

static Workspace carve(void* base, int64_t n_seq, int64_t n_tok) {
    Workspace w;
    char* p = (char*)base;
    auto take = [&](size_t bytes) { char* q = p; p += ALIGN256(bytes); return q; };
    w.part = (double*)take(8 * (size_t)(n_tok > 0 ? n_seq * n_tok : n_seq));
    w.sums = (double*)take(8 * TOTAL_GRID);
    w.totals = (int*)take(8);
    w.seq_len = (int*)take(4 * (size_t)n_seq);
    w.lp64 = (double*)take(8 * (size_t)(n_seq * n_tok));
    w.seeds = (float*)take(4 * (size_t)n_seq);
    w.stats = (RowStats*)take(sizeof(RowStats) * (size_t)(n_seq * n_tok));
    const size_t few = (size_t)(n_seq * n_tok < SPLIT_ROWS ? n_seq * n_tok : SPLIT_ROWS);
    w.acc = (Acc*)take(sizeof(Acc) * few * SPLIT_PARTS);
    w.teach = (int*)take(4 * (few < 64 ? few : 64) * TEACHER_WORDS);
    w.bytes = (size_t)(p - (char*)base);
    return w;
}

extern "C" size_t ppo_token_workspace_bytes(int64_t n_seq, int64_t n_tok) {
    if (n_seq < 0 || n_tok < 0 || n_seq > PPO_MAX_TOKENS || (n_tok > 0 && n_seq > PPO_MAX_TOKENS / n_tok)) return 0;
    return carve(nullptr, n_seq, n_tok).bytes;
}

static int check_logits(const ppo_token_logits* x, const void* grad) {
    if (!x || x->n_seq < 0 || x->n_tok < 0 || x->vocab < 1) return PPO_E_BADARG;
    if (x->dtype != PPO_F32 && x->dtype != PPO_BF16 && x->dtype != PPO_F16) return PPO_E_BADARG;
    if (!(x->inv_temperature > 1e-30) || !(x->inv_temperature < 1e30)) return PPO_E_BADARG;
    if (x->vocab > PPO_MAX_VOCAB || (x->n_tok > 0 && x->n_seq > PPO_MAX_TOKENS / x->n_tok) || x->n_seq > PPO_MAX_TOKENS)
        return PPO_E_UNSUPPORTED;
    const int64_t n = x->n_seq * x->n_tok;
    if (n == 0) return 0;
    const uintptr_t size = x->dtype == PPO_F32 ? 4 : 2;
    if (!x->data || (uintptr_t)x->data % size || (uintptr_t)grad % size) return PPO_E_BADARG;
    if (grad) {               // rows of the gradient must not overlap
        // positions within sequences or sequences within positions (a dimension of one row has no stride)
        const int64_t s = x->n_seq > 1 ? x->grad_seq_stride : INT64_MAX, t = x->n_tok > 1 ? x->grad_tok_stride : INT64_MAX;
        const int64_t inner = s < t ? s : t, outer = s < t ? t : s, many = s < t ? x->n_seq : x->n_tok;
        if (inner < x->vocab || (outer != INT64_MAX && (outer - x->vocab) / inner < many - 1)) return PPO_E_BADARG;
    }
    return 0;
}

static Logits logits_of(const ppo_token_logits* x, void* grad) {
    Logits L;
    L.x = x->data;
    L.grad = grad;
    L.xs = x->seq_stride;
    L.xt = x->tok_stride;
    L.gs = x->grad_seq_stride;
    L.gt = x->grad_tok_stride;
    L.n_tok = x->n_tok;
    L.n = x->n_seq * x->n_tok;
    L.r0 = 0;
    L.V = (int)x->vocab;
    L.c = (float)x->inv_temperature;
    L.c2 = (float)(x->inv_temperature / LN2_D);
    L.ln2 = x->inv_temperature / (double)L.c2;
    // A gradient that the 256 MB cache cannot hold is stored past it: 32768 bf16 logits a row, loss and gradient and a
    // copy of the gradient after it take 200 us against 208 at 256 MB, but 99 against 81 at 128 MB.
    L.past = L.n * L.V * (x->dtype == PPO_F32 ? 4 : 2) > (int64_t)192 << 20;
    return L;
}

#define BY_TYPE(dtype, T, ...)                                                     \
    if ((dtype) == PPO_F32) { using T = float; __VA_ARGS__; }                      \
    else if ((dtype) == PPO_BF16) { using T = __bf16; __VA_ARGS__; }               \
    else { using T = _Float16; __VA_ARGS__; }
#define BY_FLAG(flag, F, ...)                                                      \
    if (flag) { constexpr bool F = true; __VA_ARGS__; }                            \
    else { constexpr bool F = false; __VA_ARGS__; }

static int64_t row_bytes(const Logits& L, int dtype) { return (int64_t)L.V * (dtype == PPO_F32 ? 4 : 2); }

// Lanes of a row of so few logits that several share a wave; 0: more than that.  One lane's accesses are as far apart as
// the rows: 524288 rows, log-probabilities and loss with gradient, in us with one lane / with four: of 6 logits 7 / 18 and
// 21 / 36, of 8 12 / 17 and 30 / 34, of 12 10 / 18 and 40 / 35, of 16 20 / 17 and 64 / 36.
static int tiny_lanes(const Logits& L) { return L.V <= 8 ? 1 : L.V <= 64 ? 4 : L.V <= 256 ? 16 : 0; }
#define BY_LANES(lanes, G, ...)                                                    \
    if ((lanes) == 1) { constexpr int G = 1; __VA_ARGS__; }                        \
    else if ((lanes) == 4) { constexpr int G = 4; __VA_ARGS__; }                   \
    else { constexpr int G = 16; __VA_ARGS__; }

// A wave takes a row of up to 4 KB by itself: its 64 lanes hold that in four vectors each.
static bool by_wave(const Logits& L, int dtype) { return row_bytes(L, dtype) <= 4096; }

#define SOLO_ROWS 16

// A launch takes LAUNCH_ROWS rows at most: a grid of 2^32 threads and more is refused.  Runs its arguments for each
// launch with the rows' first in L.r0 and `grid` workgroups of a row, or of four (WAVE).
#define LAUNCH_ROWS (1 << 21)
#define EACH_LAUNCH(L, WAVE, grid, ...)                                            \
    for (L.r0 = 0; L.r0 < L.n; L.r0 += LAUNCH_ROWS) {                              \
        const int rows_ = (int)(L.n - L.r0 < LAUNCH_ROWS ? L.n - L.r0 : LAUNCH_ROWS); \
        const int grid = WAVE ? (rows_ + 3) / 4 : rows_;                           \
        __VA_ARGS__;                                                               \
    }

#define EACH_TINY(L, G, grid, ...) EACH_LAUNCH(L, false, rows, { const int grid = (rows + 256 / G - 1) / (256 / G); __VA_ARGS__; })

// Threads of a row that is only read: few, because what is done once a row costs each wave the same, and the chip is
// full with 512 rows under way and more (16384 rows of 16 KB: 48 us with 128 threads, 60 with 256; 4096 rows of 100 KB: 74 and
// 71); all that a workgroup can have where there are fewer rows than that.
static int stream_mode(const Logits& L, int dtype) { return by_wave(L, dtype) ? MODE_WAVE : L.n >= 512 ? MODE_BLOCK : MODE_FEW; }
static int stream_threads(const Logits& L, int dtype, int mode) {
    return mode == MODE_FEW ? 1024 : mode == MODE_BLOCK && row_bytes(L, dtype) <= 16384 ? 128 : 256;
}
#define BY_MODE(mode, M, ...)                                                      \
    if ((mode) == MODE_WAVE) { constexpr int M = MODE_WAVE; __VA_ARGS__; }         \
    else if ((mode) == MODE_BLOCK) { constexpr int M = MODE_BLOCK; __VA_ARGS__; }  \
    else { constexpr int M = MODE_FEW; __VA_ARGS__; }

// Pieces of a row where there are so few long ones (at most `rows`, of `bytes` at least) that they leave most of the chip
// idle; 0: the row is not cut.  For log-probabilities (preference's among them) and the losses that write their gradient.  Device time of bf16 rows of 256 KB, whole / cut, in us: policy loss with gradient 1 row
// 20 / 7.4, 16 rows 22 / 10, 128 rows 29 / 24 (100 KB: 12 / 7.6, 15 / 10, 18 / 15; 32 KB: no gain); distillation 1 row 20 / 10,
// 64 rows 26 / 19, 128 rows 29 / 32; log-probabilities 1 row 11 / 5.5, 64 rows 12 / 9, 256 rows 17 / 17.
static int split_parts(const Logits& L, int dtype, int64_t rows, int64_t bytes) {
    if (L.n > rows || row_bytes(L, dtype) < bytes) return 0;
    const int64_t most = row_bytes(L, dtype) / 8192, want = 1024 / L.n;
    const int64_t parts = want < most ? want : most;
    return (int)(parts < SPLIT_PARTS ? parts : SPLIT_PARTS);
}

// Threads of a row that is held in CH vectors each: as many as it needs (a shift may leave up to 7
// vectors over, which are read twice).
static int held_threads(const Logits& L, int dtype, int CH) {
    const int64_t waves = (row_bytes(L, dtype) + (int64_t)CH * 16 * 64 - 1) / ((int64_t)CH * 16 * 64);
    return (int)(waves < 16 ? waves : 16) * 64;
}
// 8 vectors a thread for rows of up to 96 KB, else 16 (4096 rows with their gradient: of 80 KB 122 us against 131 with 16,
// of 100 KB 187 against 161); the rest of a row beyond 256 KB is read twice.
static bool held_in_8(const Logits& L, int dtype) { return row_bytes(L, dtype) <= 96 * 1024; }

static void launch_total(const Workspace& w, int64_t n, float* loss, hipStream_t st) {
    if (n <= 16384) {
        total_kernel<<<1, 1024, 0, st>>>(w.part, n, nullptr, loss);
        return;
    }
    total_kernel<<<TOTAL_GRID, 1024, 0, st>>>(w.part, n, w.sums, nullptr);
    total_kernel<<<1, 1024, 0, st>>>(w.sums, TOTAL_GRID, nullptr, loss);
}

// Counted rows of each sequence and of all, where a weight needs them.
static void count_rows(const Weights& o, const ppo_token_logits* x, const Workspace& w, hipStream_t st) {
    const uint8_t* mask = o.mask;
    if (!mask || o.reduction == RED_SUM || o.count_here) return;
    if (x->n_seq * x->n_tok <= 32768) {
        count_kernel<<<1, 1024, 0, st>>>(mask, x->n_seq, x->n_tok, w.seq_len, w.totals, 1, 1);
        return;
    }
    const int64_t g = (x->n_seq + 15) / 16;
    count_kernel<<<(int)(g < 1024 ? g : 1024), 1024, 0, st>>>(mask, x->n_seq, x->n_tok, w.seq_len, w.totals, 1, 0);
    count_kernel<<<1, 1024, 0, st>>>(mask, x->n_seq, x->n_tok, w.seq_len, w.totals, 0, 1);
}

static int weights_of(Weights* o, const uint8_t* mask, int reduction, float scale, const ppo_token_logits* x,
                      const Workspace& w) {
    if (reduction != RED_SUM && reduction != RED_TOKEN && reduction != RED_SEQ) return PPO_E_BADARG;
    const int here = mask && reduction != RED_SUM && x->n_seq * x->n_tok <= COUNT_HERE &&
                     (reduction == RED_TOKEN || x->n_seq <= COUNT_SEQS);
    *o = {mask, w.seq_len, w.totals, reduction, here, scale, x->n_seq};
    return 0;
}

// logprobs64, which are summed over a sequence and compared, are computed with E: what ln_sum takes back with it is up to
// 1e-7 a token, the same way in all of them.
static void launch_logprobs(Logits L, int dtype, const void* tokens, int i64, const uint8_t* mask, float* logprobs,
                            double* logprobs64, float* entropy, RowStats* stats, Acc* acc, hipStream_t st) {
    const bool with_e = entropy || logprobs64;
    if (const int parts = acc ? split_parts(L, dtype, PPO_TOKEN_CUT_ROWS, PPO_TOKEN_CUT_BYTES) : 0) {
        const Split sp = {acc, nullptr, parts};
        BY_FLAG(with_e, ENT, {
            BY_TYPE(dtype, T, (split_stats_kernel<T, ENT><<<dim3((unsigned)L.n, parts), 256, 0, st>>>(L, mask, tokens, i64, sp)))
            split_logprobs_kernel<ENT><<<(int)(L.n + 3) / 4, 256, 0, st>>>(L, mask, logprobs, logprobs64, entropy, stats, sp);
        })
        return;
    }
    if (const int lanes = tiny_lanes(L)) {
        BY_TYPE(dtype, T, BY_LANES(lanes, G, EACH_TINY(L, G, grid, (tiny_logprobs_kernel<T, G><<<grid, 256, 0, st>>>(
            L, tokens, i64, mask, logprobs, logprobs64, entropy, stats)))))
        return;
    }
    BY_TYPE(dtype, T, BY_MODE(stream_mode(L, dtype), MODE, BY_FLAG(with_e, ENT, BY_FLAG(stats != nullptr, KEEP, {
        EACH_LAUNCH(L, MODE == MODE_WAVE, grid, (logprobs_kernel<T, MODE, ENT, KEEP><<<grid, stream_threads(L, dtype, MODE), 0, st>>>(
            L, tokens, i64, mask, logprobs, logprobs64, entropy, stats)))
    }))))
}

// Threads of a row in the backward pass: 1024 of long rows (rows of 64 KB: 127 us against 134 with 256), 256 of rows that
// would leave them without work (rows of 8 KB: 83 us against 128).
static int backward_threads(const Logits& L, int dtype) { return row_bytes(L, dtype) >= 32768 ? 1024 : 256; }

// Parts of a row that the backward pass gives to a workgroup each, so that few rows fill the chip too: at least 64 KB.
static int backward_parts(const Logits& L, int dtype) {
    const int64_t want = (1024 + L.n - 1) / L.n, most = (row_bytes(L, dtype) + 65535) / 65536;
    return (int)(want < most ? want : most);
}

extern "C" int ppo_token_logprobs(const ppo_token_logits* x, const void* tokens, int tokens_are_i64,
                                  const uint8_t* mask, float* logprobs, float* entropy, float* row_stats, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    const int e = check_logits(x, nullptr);
    if (e) return e;
    Logits L = logits_of(x, nullptr);
    if (L.n == 0) return 0;
    if (!tokens || !logprobs) return PPO_E_BADARG;
    const Workspace w = carve(workspace, x->n_seq, x->n_tok);
    if (workspace && workspace_bytes < w.bytes) return PPO_E_WORKSPACE;
    if ((uintptr_t)workspace % 16) return PPO_E_BADARG;
    launch_logprobs(L, x->dtype, tokens, tokens_are_i64, mask, logprobs, nullptr, entropy, (RowStats*)row_stats,
                    workspace ? w.acc : nullptr, (hipStream_t)stream);
    return (int)hipGetLastError();
}

static int launch_backward(Logits L, int dtype, const void* tokens, int i64, const uint8_t* mask,
                           const RowStats* stats, const Incoming& in, hipStream_t st) {
    if (const int lanes = tiny_lanes(L)) {
        BY_TYPE(dtype, T, BY_LANES(lanes, G, EACH_TINY(L, G, grid, (tiny_backward_kernel<T, G><<<grid, 256, 0, st>>>(
            L, tokens, i64, mask, stats, in)))))
        return (int)hipGetLastError();
    }
    BY_TYPE(dtype, T, BY_FLAG(by_wave(L, dtype), WAVE, BY_FLAG(in.h != nullptr, ENT, {
        EACH_LAUNCH(L, WAVE, grid, (backward_kernel<T, WAVE, ENT><<<dim3(grid, WAVE ? 1 : backward_parts(L, dtype)), WAVE ? 256 : backward_threads(L, dtype), 0, st>>>(
            L, tokens, i64, mask, stats, in)))
    })))
    return (int)hipGetLastError();
}

extern "C" int ppo_token_logprobs_backward(const ppo_token_logits* x, const void* tokens, int tokens_are_i64,
                                           const uint8_t* mask, const float* row_stats, const float* grad_logprobs,
                                           int64_t lp_seq_stride, int64_t lp_tok_stride, const float* grad_entropy,
                                           int64_t ent_seq_stride, int64_t ent_tok_stride, const float* grad_factor,
                                           void* grad, void* stream) {
    const int e = check_logits(x, grad);
    if (e) return e;
    Logits L = logits_of(x, grad);
    if (L.n == 0) return 0;
    if (!tokens || !row_stats || !grad) return PPO_E_BADARG;
    const Incoming in = {grad_logprobs, grad_entropy, grad_factor, lp_seq_stride, lp_tok_stride, ent_seq_stride,
                         ent_tok_stride};
    return launch_backward(L, x->dtype, tokens, tokens_are_i64, mask, (const RowStats*)row_stats, in, (hipStream_t)stream);
}

extern "C" int ppo_policy_loss(const ppo_token_logits* x, const void* tokens, int tokens_are_i64, const uint8_t* mask,
                               const float* old_logprobs, const float* advantages, int64_t adv_seq_stride,
                               int64_t adv_tok_stride, const float* ref_logprobs, const ppo_policy_terms* terms,
                               float* loss, float* logprobs, float* entropy, float* row_stats, float* seeds,
                               void* grad, void* workspace, size_t workspace_bytes, void* stream) {
    int e = check_logits(x, grad);
    if (e) return e;
    if (!terms || !loss || (terms->kl_coef != 0.0f && !ref_logprobs) || (row_stats && !seeds)) return PPO_E_BADARG;
    const hipStream_t st = (hipStream_t)stream;
    const Workspace w = carve(workspace, x->n_seq, x->n_tok);
    if (!workspace || workspace_bytes < w.bytes) return PPO_E_WORKSPACE;
    if ((uintptr_t)workspace % 16) return PPO_E_BADARG;
    Logits L = logits_of(x, grad);
    PolicyArgs p;
    bool solo = false;
    e = weights_of(&p.w, mask, terms->reduction, terms->scale, x, w);
    if (e) return e;
    if (L.n > 0) {
        if (!tokens || !old_logprobs || !advantages || !logprobs) return PPO_E_BADARG;
        p.tokens = tokens;
        p.i64 = tokens_are_i64;
        p.old_lp = old_logprobs;
        p.adv = advantages;
        p.adv_s = adv_seq_stride;
        p.adv_t = adv_tok_stride;
        p.ref = ref_logprobs;
        p.lo = 1.0f - terms->clip_low;
        p.hi = 1.0f + terms->clip_high;
        p.kl = terms->kl_coef;
        p.ent = terms->entropy_coef;
        p.logprobs = logprobs;
        p.entropy = entropy;
        p.stats = (RowStats*)row_stats;
        p.g_lp = seeds;
        p.g_h = seeds ? seeds + L.n : nullptr;
        p.part = w.part;
        // One workgroup, of a wave for each row, where that takes them all: the loss then needs no second launch.
        const int lanes = tiny_lanes(L);
        solo = L.n == 1 || (!lanes && by_wave(L, x->dtype) && L.n <= SOLO_ROWS);
        p.solo = solo ? loss : nullptr;
        if (lanes) p.w.count_here = 0;
        count_rows(p.w, x, w, st);
        if (lanes) {
            BY_TYPE(x->dtype, T, BY_LANES(lanes, G, BY_FLAG(grad != nullptr, GRAD, {
                EACH_TINY(L, G, grid, (tiny_policy_kernel<T, G, GRAD><<<grid, 256, 0, st>>>(L, p)))
            })))
        } else if (!grad) {
            BY_TYPE(x->dtype, T, BY_MODE(stream_mode(L, x->dtype), MODE, {
                const int threads = solo && MODE == MODE_WAVE ? 64 * (int)L.n : stream_threads(L, x->dtype, MODE);
                EACH_LAUNCH(L, MODE == MODE_WAVE, grid, (policy_forward_kernel<T, MODE><<<solo ? 1 : grid, threads, 0, st>>>(L, p)))
            }))
        } else if (const int parts = split_parts(L, x->dtype, 128, 64 * 1024)) {
            const Split sp = {w.acc, nullptr, parts};
            const dim3 grid((unsigned)L.n, parts);
            BY_TYPE(x->dtype, T, BY_FLAG(p.ent != 0.0f, ENT, {
                split_stats_kernel<T, true><<<grid, 256, 0, st>>>(L, mask, tokens, tokens_are_i64, sp);
                policy_split_kernel<T, ENT><<<grid, 256, 0, st>>>(L, p, sp);
            }))
        } else {
            BY_TYPE(x->dtype, T, BY_FLAG(p.ent != 0.0f, ENT, {
                if (by_wave(L, x->dtype))
                    EACH_LAUNCH(L, true, grid, (policy_kernel<T, 4, true, ENT><<<solo ? 1 : grid, solo ? 64 * (int)L.n : 256, 0, st>>>(L, p)))
                else if (held_in_8(L, x->dtype))
                    EACH_LAUNCH(L, false, grid, (policy_kernel<T, 8, false, ENT><<<grid, held_threads(L, x->dtype, 8), 0, st>>>(L, p)))
                else
                    EACH_LAUNCH(L, false, grid, (policy_kernel<T, 16, false, ENT><<<grid, held_threads(L, x->dtype, 16), 0, st>>>(L, p)))
            }))
        }
    }
    if (!solo) launch_total(w, L.n, loss, st);
    return (int)hipGetLastError();
}

extern "C" int ppo_preference_loss(const ppo_token_logits* x, const void* tokens, int tokens_are_i64,
                                   const uint8_t* mask, const float* ref_logprobs, double beta, double label_smoothing,
                                   double scale, float* loss, float* rewards, float* row_stats, float* seeds,
                                   void* grad, void* workspace, size_t workspace_bytes, void* stream) {
    const int e = check_logits(x, grad);
    if (e) return e;
    if (x->n_seq < 2 || x->n_seq % 2 || !loss || !rewards || !ref_logprobs || (row_stats && !seeds)) return PPO_E_BADARG;
    const hipStream_t st = (hipStream_t)stream;
    const Workspace w = carve(workspace, x->n_seq, x->n_tok);
    if (!workspace || workspace_bytes < w.bytes) return PPO_E_WORKSPACE;
    if ((uintptr_t)workspace % 16) return PPO_E_BADARG;
    Logits L = logits_of(x, grad);
    if (L.n > 0 && !tokens) return PPO_E_BADARG;
    const int64_t pairs = x->n_seq / 2;
    RowStats* stats = row_stats ? (RowStats*)row_stats : w.stats;
    float* sd = seeds ? seeds : w.seeds;
    if (L.n > 0) {
        launch_logprobs(L, x->dtype, tokens, tokens_are_i64, mask, nullptr, w.lp64, nullptr, stats, w.acc, st);
    }
    pair_kernel<<<(int)(pairs < LAUNCH_ROWS ? pairs : LAUNCH_ROWS), 256, 0, st>>>(w.lp64, mask, ref_logprobs, pairs, x->n_tok, beta, label_smoothing, scale,
                                                rewards, sd, w.part, pairs == 1 ? loss : nullptr);
    if (pairs > 1) launch_total(w, pairs, loss, st);
    if (grad && L.n > 0) {
        const Incoming in = {sd, nullptr, nullptr, 1, 0, 0, 0};
        return launch_backward(L, x->dtype, tokens, tokens_are_i64, mask, stats, in, st);
    }
    return (int)hipGetLastError();
}

static int teacher_of(TeacherArgs* p, const ppo_token_logits* x, const void* index, int i64, const void* logit, int dtype,
                      int K) {
    if (K < 1) return PPO_E_BADARG;
    if (K > PPO_MAX_TEACHER_TOP) return PPO_E_UNSUPPORTED;
    if (dtype != PPO_F32 && dtype != PPO_BF16 && dtype != PPO_F16) return PPO_E_BADARG;
    if (x->n_seq * x->n_tok > 0 && (!index || !logit)) return PPO_E_BADARG;
    *p = {};
    p->index = index;
    p->logit = logit;
    p->i64 = i64;
    p->dtype = dtype;
    p->K = K;
    return 0;
}

extern "C" int ppo_distillation_loss(const ppo_token_logits* x, const void* teacher_tokens, int tokens_are_i64,
                                     const void* teacher_logits, int teacher_dtype, int top, const uint8_t* mask,
                                     int reduction, float scale, float* loss, float* token_losses, float* row_stats,
                                     void* grad, void* workspace, size_t workspace_bytes, void* stream) {
    int e = check_logits(x, grad);
    TeacherArgs p;
    if (!e) e = teacher_of(&p, x, teacher_tokens, tokens_are_i64, teacher_logits, teacher_dtype, top);
    if (e) return e;
    if (!loss) return PPO_E_BADARG;
    const hipStream_t st = (hipStream_t)stream;
    const Workspace w = carve(workspace, x->n_seq, x->n_tok);
    if (!workspace || workspace_bytes < w.bytes) return PPO_E_WORKSPACE;
    if ((uintptr_t)workspace % 16) return PPO_E_BADARG;
    e = weights_of(&p.w, mask, reduction, scale, x, w);
    if (e) return e;
    Logits L = logits_of(x, grad);
    p.losses = token_losses;
    p.stats = (RowStats*)row_stats;
    p.part = w.part;
    p.solo = L.n == 1 ? loss : nullptr;
    if (L.n > 0) {
        count_rows(p.w, x, w, st);
        const size_t lds = teacher_lds(top);
        const int parts = grad ? split_parts(L, x->dtype, 64, 128 * 1024) : 0;
        const Split sp = {w.acc, w.teach, parts};
        BY_TYPE(x->dtype, T, {
            if (!grad && L.n >= 512)
                EACH_LAUNCH(L, false, grid, (distill_forward_kernel<T, MODE_BLOCK><<<grid, stream_threads(L, x->dtype, MODE_BLOCK), lds, st>>>(L, p)))
            else if (!grad)
                EACH_LAUNCH(L, false, grid, (distill_forward_kernel<T, MODE_FEW><<<grid, stream_threads(L, x->dtype, MODE_FEW), lds, st>>>(L, p)))
            else if (parts) {
                const dim3 grid((unsigned)L.n, parts);
                split_teacher_kernel<T><<<dim3((unsigned)L.n, parts + 1), 256, lds, st>>>(L, p, sp);
                distill_split_kernel<T><<<grid, 256, lds, st>>>(L, p, sp);
            } else if (held_in_8(L, x->dtype))
                EACH_LAUNCH(L, false, grid, (distill_kernel<T, 8><<<grid, held_threads(L, x->dtype, 8), lds, st>>>(L, p)))
            else
                EACH_LAUNCH(L, false, grid, (distill_kernel<T, 16><<<grid, held_threads(L, x->dtype, 16), lds, st>>>(L, p)))
        })
    }
    if (L.n != 1) launch_total(w, L.n, loss, st);
    return (int)hipGetLastError();
}

extern "C" int ppo_distillation_backward(const ppo_token_logits* x, const void* teacher_tokens, int tokens_are_i64,
                                         const void* teacher_logits, int teacher_dtype, int top, const uint8_t* mask,
                                         const float* row_stats, const float* grad_factor, void* grad, void* stream) {
    int e = check_logits(x, grad);
    TeacherArgs p;
    if (!e) e = teacher_of(&p, x, teacher_tokens, tokens_are_i64, teacher_logits, teacher_dtype, top);
    if (e) return e;
    Logits L = logits_of(x, grad);
    if (L.n == 0) return 0;
    if (!row_stats || !grad) return PPO_E_BADARG;
    p.w.mask = mask;
    p.stats = (RowStats*)row_stats;
    p.factor = grad_factor;
    BY_TYPE(x->dtype, T, EACH_LAUNCH(L, false, grid, (distill_backward_kernel<T><<<grid, backward_threads(L, x->dtype), teacher_lds(top), (hipStream_t)stream>>>(L, p))))
    return (int)hipGetLastError();
}
