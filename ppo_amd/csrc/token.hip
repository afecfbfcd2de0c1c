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
// product on each e_i.  u_i is formed as a difference first: it is 0 at the maximum for any size of the logits
// (c x - c m would leave the rounding of a large c m), and a logit of -inf or of the type's lowest value has
// e_i = 0.  Sums are fp32 within a thread and over the workgroup, one row's scalars are finished in fp64.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ppo_hip.h"

#define LOG2E_F 1.4426950408889634f
#define LN2_D 0.6931471805599453
#define U_FLOOR (-1.0e6f)    // below it e_i is 0: products e_i u_i take this in place of -inf
#define MAX_GRID 8192        // workgroups of a launch; rows beyond are taken in turns

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

template <typename T> __device__ __forceinline__ u32x4 load_vec(const T* p) {   // p: aligned for T only
    u32x4 o;
    __builtin_memcpy(&o, p, 16);
    return o;
}
template <typename T> __device__ __forceinline__ void store_vec(T* p, u32x4 o) { __builtin_memcpy(p, &o, 16); }

// This thread's vector of the vectors that begin at a uniform address: one 32-bit offset for all
// of a thread's accesses, the rest in scalar registers.
template <typename T> __device__ __forceinline__ u32x4 load_at(const T* base) {
    return load_vec((const T*)((const char*)base + threadIdx.x * 16u));
}
template <typename T> __device__ __forceinline__ void store_at(T* base, u32x4 o) {
    store_vec((T*)((char*)base + threadIdx.x * 16u), o);
}

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
};

__device__ __forceinline__ Acc acc_empty() { return {-__FLT_MAX__, 0.0f, 0.0f}; }   // finite: -inf logits give u = -inf

// a, relative to a larger maximum mn
template <bool ENT> __device__ __forceinline__ void acc_rebase(Acc& a, float mn, float c2) {
    const float d = fmaxf((a.m - mn) * c2, -1.0e30f);
    const float r = __builtin_amdgcn_exp2f(d);
    if (ENT) a.e = (a.e + a.s * d) * r;
    a.s *= r;
    a.m = mn;
}

template <bool ENT> __device__ __forceinline__ void acc_add(Acc& a, float x, float c2) {   // a.m >= x, or x is NaN
    const float u = (x - a.m) * c2;
    const float e = __builtin_amdgcn_exp2f(u);
    a.s += e;
    if (ENT) a.e = fmaf(e, fmaxf(u, U_FLOOR), a.e);
}

// 16 * M bytes of logits at once: their maximum, one rescaling, their terms
template <typename T, int M, bool ENT> __device__ __forceinline__ void acc_vecs(Acc& a, const u32x4* v, float c2) {
    constexpr int N = VEC<T>;
    float f[N * M], mx = a.m;
#pragma unroll
    for (int k = 0; k < M; ++k) unpack<T>(v[k], f + k * N);
#pragma unroll
    for (int i = 0; i < N * M; ++i) mx = fmaxf(mx, f[i]);
    acc_rebase<ENT>(a, mx, c2);
#pragma unroll
    for (int i = 0; i < N * M; ++i) acc_add<ENT>(a, f[i], c2);
}

// Rotation within the 16 lanes of a row: an all-reduce in four steps without LDS.  Partners add the same two
// numbers, so all lanes end with the same bits.
template <int CTRL> __device__ __forceinline__ float ror(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float lane_value(float x, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}
template <int W> __device__ __forceinline__ float row_max(float x) {   // of W = 1, 2, 4, 8, 16 lanes' values
    if (W > 8) x = fmaxf(x, ror<0x128>(x));
    if (W > 4) x = fmaxf(x, ror<0x124>(x));
    if (W > 2) x = fmaxf(x, ror<0x122>(x));
    if (W > 1) x = fmaxf(x, ror<0x121>(x));
    return x;
}
template <int W> __device__ __forceinline__ float row_sum(float x) {
    if (W > 8) x += ror<0x128>(x);
    if (W > 4) x += ror<0x124>(x);
    if (W > 2) x += ror<0x122>(x);
    if (W > 1) x += ror<0x121>(x);
    return x;
}
__device__ __forceinline__ float wave_max(float x) {
    x = row_max<16>(x);
    return fmaxf(fmaxf(lane_value(x, 0), lane_value(x, 16)), fmaxf(lane_value(x, 32), lane_value(x, 48)));
}
__device__ __forceinline__ float wave_sum(float x) {
    x = row_sum<16>(x);
    return (lane_value(x, 0) + lane_value(x, 16)) + (lane_value(x, 32) + lane_value(x, 48));
}

// The threads' accumulators joined; every thread returns the same bits.  lds: NT / 64 entries.
template <int NT, bool ENT> __device__ __forceinline__ Acc acc_block(Acc a, float c2, Acc* lds) {
    constexpr int W = NT / 64;
    acc_rebase<ENT>(a, wave_max(a.m), c2);
    a.s = wave_sum(a.s);
    if (ENT) a.e = wave_sum(a.e);
    if (W == 1) return a;
    __syncthreads();          // the previous row's values have been read
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
    __syncthreads();
    a = lds[threadIdx.x & (W - 1)];
    acc_rebase<ENT>(a, row_max<W>(a.m), c2);
    a.s = lane_value(row_sum<W>(a.s), 0);
    if (ENT) a.e = lane_value(row_sum<W>(a.e), 0);
    a.m = lane_value(a.m, 0);
    return a;
}

// ------------------------------------------------------------------------------------------ a row on the chip
// NT threads hold up to NT * HELD * 16 bytes of a row in registers, so that statistics and gradient read memory
// once; the vectors beyond are read again for the gradient.  Vector j belongs to thread j % NT.  Vectors past the
// end are filled with -inf, which adds nothing; the V % N last logits are one scalar of as many threads.
#define HELD 16

template <typename T, int NT> struct Row {
    static constexpr int N = VEC<T>;
    u32x4 v[HELD];
    T tail;

    __device__ __forceinline__ void load(const T* x, int V) {
        const int nvec = V / N;
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            v[i] = Word<T>::LOWEST;
            if ((int)threadIdx.x < nvec - i * NT) v[i] = load_at(x + i * NT * N);
        }
        tail = (T)-__builtin_inff();
        if ((int)threadIdx.x < V - nvec * N) tail = x[nvec * N + threadIdx.x];
    }
};

// vectors joined before each rescaling
template <typename T> struct Step { static constexpr int M = sizeof(T) == 4 ? 4 : 2; };

template <typename T, int NT, bool ENT>
__device__ __forceinline__ Acc row_stats(const Row<T, NT>& row, const T* x, int V, float c2, Acc* lds) {
    constexpr int N = VEC<T>, M = Step<T>::M;
    const int nvec = V / N;
    Acc a = acc_empty();
#pragma unroll
    for (int i = 0; i < HELD; i += M) {
        if (i * NT >= nvec) break;
        acc_vecs<T, M, ENT>(a, row.v + i, c2);
    }
    if (NT == 1024)
        for (int j = HELD * NT + threadIdx.x; j < nvec; j += NT) {
            const u32x4 v = load_vec(x + (int64_t)j * N);
            acc_vecs<T, 1, ENT>(a, &v, c2);
        }
    const float t = wide(row.tail);
    acc_rebase<ENT>(a, fmaxf(a.m, t), c2);
    acc_add<ENT>(a, t, c2);
    return acc_block<NT, ENT>(a, c2, lds);
}

// ------------------------------------------------------------------------------------------ row gradient
// dL/dx_i = e_i (a + b u_i), + gt at `tok`
struct RowGrad {
    float m, a, b, gt;
    int tok;     // -1: none
};

template <bool ENT> __device__ __forceinline__ float grad_of(const RowGrad& g, float x, float c2) {
    const float u = (x - g.m) * c2;
    const float e = __builtin_amdgcn_exp2f(u);
    return ENT ? e * fmaf(g.b, fmaxf(u, U_FLOOR), g.a) : e * g.a;
}

template <typename T, bool ENT>
__device__ __forceinline__ u32x4 grad_vec(const RowGrad& g, u32x4 v, int j, float c2) {
    constexpr int N = VEC<T>;
    float d[N];
    unpack<T>(v, d);
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = grad_of<ENT>(g, d[i], c2);
    if (j == g.tok / N && g.tok >= 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] += i == g.tok % N ? g.gt : 0.0f;
    }
    return pack<T>(d);        // the one rounding of the gradient
}

template <typename T, bool ENT> __device__ __forceinline__ T grad_one(const RowGrad& g, T x, int i, float c2) {
    const float d = grad_of<ENT>(g, wide(x), c2);
    return (T)(i == g.tok ? d + g.gt : d);
}

// the gradient of a held row; the vectors that are read again may lie where the gradient goes
template <typename T, int NT, bool ENT>
__device__ __forceinline__ void row_grad(const Row<T, NT>& row, const T* x, T* out, int V, float c2, const RowGrad& g) {
    constexpr int N = VEC<T>;
    const int nvec = V / N;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        if (i * NT >= nvec) break;
        const u32x4 o = grad_vec<T, ENT>(g, row.v[i], i * NT + threadIdx.x, c2);
        if ((int)threadIdx.x < nvec - i * NT) store_at(out + i * NT * N, o);
    }
    if (NT == 1024)
        for (int j = HELD * NT + threadIdx.x; j < nvec; j += NT)
            store_vec(out + (int64_t)j * N, grad_vec<T, ENT>(g, load_vec(x + (int64_t)j * N), j, c2));
    const int i = nvec * N + threadIdx.x;
    if (i < V) out[i] = grad_one<T, ENT>(g, row.tail, i, c2);
}

// the gradient of a row whose statistics are known; x may be out
template <typename T, int NT, bool ENT>
__device__ __forceinline__ void row_map(const T* x, T* out, int V, float c2, const RowGrad& g) {
    constexpr int N = VEC<T>;
    const int nvec = V / N;
    for (int j = threadIdx.x; j < nvec; j += NT)
        store_vec(out + (int64_t)j * N, grad_vec<T, ENT>(g, load_vec(x + (int64_t)j * N), j, c2));
    for (int i = nvec * N + threadIdx.x; i < V; i += NT) out[i] = grad_one<T, ENT>(g, x[i], i, c2);
}

template <typename T, int NT> __device__ __forceinline__ void row_fill(T* out, int V, float value) {
    constexpr int N = VEC<T>;
    const int nvec = V / N;
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = value;
    const u32x4 o = pack<T>(f);
    for (int j = threadIdx.x; j < nvec; j += NT) store_vec(out + (int64_t)j * N, o);
    for (int i = nvec * N + threadIdx.x; i < V; i += NT) out[i] = (T)value;
}

// ------------------------------------------------------------------------------------------ launch arguments
struct Logits {
    const void* x;
    void* grad;               // may be x itself
    int64_t xs, xt, gs, gt;   // strides (elements) of sequences and tokens
    int64_t n_tok, n;         // n = sequences * n_tok rows
    int V;
    float c, c2;              // 1/temperature; the same times log2(e)
};

template <typename T> __device__ __forceinline__ const T* row_in(const Logits& L, int64_t b, int64_t t) {
    return (const T*)L.x + b * L.xs + t * L.xt;
}
template <typename T> __device__ __forceinline__ T* row_out(const Logits& L, int64_t b, int64_t t) {
    return (T*)L.grad + b * L.gs + t * L.gt;
}

struct Weights {              // how much a row counts
    const uint8_t* mask;      // NULL: every row counts
    const int* seq_len;       // counted rows of each sequence (masks only)
    const int* totals;        // {counted rows, sequences with one} (masks only)
    int reduction;
    float scale;
    int64_t n_seq;
};

__device__ __forceinline__ float row_weight(const Weights& w, int64_t b, int64_t n_tok) {   // of a counted row
    double d = 1.0;
    if (w.reduction == RED_TOKEN) d = w.mask ? (double)w.totals[0] : (double)w.n_seq * (double)n_tok;
    if (w.reduction == RED_SEQ)
        d = w.mask ? (double)w.seq_len[b] * (double)w.totals[1] : (double)w.n_seq * (double)n_tok;
    return (float)((double)w.scale / d);
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
    const double z = ((double)f - 1.0) / ((double)f + 1.0), y = z * z;
    const double p = fma(y, fma(y, fma(y, fma(y, fma(y, 1.0 / 11, 1.0 / 9), 1.0 / 7), 1.0 / 5), 1.0 / 3), 1.0);
    return fma((double)k, LN2_D, 2.0 * z * p);
}

// log-probability of `tok`, NaN for one that is not in the vocabulary (its row of logits is not indexed with it)
template <typename T>
__device__ __forceinline__ double token_logp(const T* x, int64_t tok, int V, float c, const Acc& a, double ln_s) {
    if (tok < 0 || tok >= V) return __builtin_nan("");
    return ((double)wide(x[tok]) - (double)a.m) * (double)c - ln_s;
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

// sum of `n` partial losses in a fixed order
__global__ __launch_bounds__(1024) void total_kernel(const double* __restrict__ part, int n, float* loss) {
    __shared__ double lds[16];
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) s += part[i];
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) s += lds[w];
        *loss = (float)s;
    }
}

// ------------------------------------------------------------------------------------------ log-probabilities
template <typename T, int NT, bool ENT>
__global__ __launch_bounds__(NT, 4) void logprobs_kernel(Logits L, const void* tokens, int i64, const uint8_t* mask,
                                                      float* logprobs, double* logprobs64, float* entropy,
                                                      RowStats* stats) {
    __shared__ Acc lds[NT / 64];
    for (int64_t r = blockIdx.x; r < L.n; r += gridDim.x) {
        const int64_t b = r / L.n_tok, t = r - b * L.n_tok;
        double lp = 0.0;
        RowStats st = {0.0f, 1.0f, 0.0f, 0.0f};
        if (!mask || mask[r]) {
            const T* x = row_in<T>(L, b, t);
            Row<T, NT> row;
            row.load(x, L.V);
            const Acc a = row_stats<T, NT, ENT>(row, x, L.V, L.c2, lds);
            const double ln_s = ln_of(a.s);
            lp = token_logp(x, int_at(tokens, i64, r), L.V, L.c, a, ln_s);
            st.m = a.m;
            st.s = a.s;
            if (ENT) st.h = (float)(ln_s - LN2_D * (double)(a.e / a.s));
        }
        if (threadIdx.x == 0) {
            if (logprobs) logprobs[r] = (float)lp;
            if (logprobs64) logprobs64[r] = lp;
            if (ENT && entropy) entropy[r] = st.h;
            if (stats) stats[r] = st;
        }
    }
}

__device__ __forceinline__ RowGrad grad_seed(float m, float s, float h, float g_lp, float g_h, int64_t tok, int V,
                                             float c) {
    RowGrad g;
    g.m = m;
    const float ln_s = (float)ln_of(s);
    const bool bad = tok < 0 || tok >= V;
    g.a = bad ? __builtin_nanf("") : -c * (g_lp + g_h * (h - ln_s)) / s;
    g.b = -c * g_h * (float)LN2_D / s;
    g.gt = c * g_lp;
    g.tok = bad ? -1 : (int)tok;
    return g;
}

struct Incoming {             // dL/dlogp and dL/dH of each row, and a factor on both
    const float *lp, *h, *factor;
    int64_t lp_s, lp_t, h_s, h_t;
};

template <typename T, int NT, bool ENT>
__global__ __launch_bounds__(NT, 4) void backward_kernel(Logits L, const void* tokens, int i64, const uint8_t* mask,
                                                      const RowStats* __restrict__ stats, Incoming in) {
    const float f = in.factor ? *in.factor : 1.0f;
    for (int64_t r = blockIdx.x; r < L.n; r += gridDim.x) {
        const int64_t b = r / L.n_tok, t = r - b * L.n_tok;
        T* out = row_out<T>(L, b, t);
        if (mask && !mask[r]) {
            row_fill<T, NT>(out, L.V, 0.0f);
            continue;
        }
        const RowStats st = stats[r];
        const float g_lp = in.lp ? f * in.lp[b * in.lp_s + t * in.lp_t] : 0.0f;
        const float g_h = ENT ? f * in.h[b * in.h_s + t * in.h_t] : 0.0f;
        const RowGrad g = grad_seed(st.m, st.s, st.h, g_lp, g_h, int_at(tokens, i64, r), L.V, L.c);
        row_map<T, NT, ENT>(row_in<T>(L, b, t), out, L.V, L.c2, g);
    }
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
    double* part;
};

struct PolicyRow {
    double loss;              // weighted, as the gradients are
    float g_lp, g_h;
};

__device__ __forceinline__ PolicyRow policy_row(const PolicyArgs& p, double lp, float h, float old_lp, float adv,
                                                float ref, float w) {
    // Differences of log-probabilities are formed in fp64, where they lose nothing.  The ratio is 1 + (e^d - 1) with
    // the second part in fp32: near 1 that keeps more of it than fp32 does, and a loss is a mean in which A and -A
    // nearly cancel.
    const double r = 1.0 + (double)expm1f((float)(lp - (double)old_lp)), a = (double)adv;
    const bool clipped = (adv > 0.0f && r > (double)p.hi) || (adv < 0.0f && r < (double)p.lo);
    double loss = clipped ? -(adv > 0.0f ? (double)p.hi : (double)p.lo) * a : -r * a;
    float g = clipped ? 0.0f : (float)(-r * a);
    if (p.kl != 0.0f) {
        const float d = (float)((double)ref - lp);
        // e^d - 1 - d: its series where the difference would cancel (|d|^6 / 20160 < 2^-24 at 1/4)
        const float em1 = expm1f(d);
        const float k = fabsf(d) < 0.25f
            ? d * d * fmaf(d, fmaf(d, fmaf(d, fmaf(d, fmaf(d, 1.0f / 5040, 1.0f / 720), 1.0f / 120), 1.0f / 24), 1.0f / 6), 0.5f)
            : em1 - d;
        loss = fma((double)p.kl, (double)k, loss);
        g = fmaf(-p.kl, em1, g);
    }
    if (p.ent != 0.0f) loss = fma(-(double)p.ent, (double)h, loss);
    return {loss * (double)w, w * g, -w * p.ent};
}

template <typename T, int NT, bool GRAD, bool ENT_GRAD>
__global__ __launch_bounds__(NT, 4) void policy_kernel(Logits L, PolicyArgs p) {
    __shared__ Acc lds[NT / 64];
    double total = 0.0;
    for (int64_t r = blockIdx.x; r < L.n; r += gridDim.x) {
        const int64_t b = r / L.n_tok, t = r - b * L.n_tok;
        RowStats st = {0.0f, 1.0f, 0.0f, 0.0f};
        double lp = 0.0;
        PolicyRow o = {0.0, 0.0f, 0.0f};
        if (!p.w.mask || p.w.mask[r]) {
            const T* x = row_in<T>(L, b, t);
            Row<T, NT> row;
            row.load(x, L.V);
            const Acc a = row_stats<T, NT, true>(row, x, L.V, L.c2, lds);
            const double ln_s = ln_of(a.s);
            const int64_t tok = int_at(p.tokens, p.i64, r);
            lp = token_logp(x, tok, L.V, L.c, a, ln_s);
            st.m = a.m;
            st.s = a.s;
            st.h = (float)(ln_s - LN2_D * (double)(a.e / a.s));
            o = policy_row(p, lp, st.h, p.old_lp[r], p.adv[b * p.adv_s + t * p.adv_t], p.ref ? p.ref[r] : 0.0f,
                           row_weight(p.w, b, L.n_tok));
            total += o.loss;
            if (GRAD) {
                __syncthreads();   // x[tok] has been read by all: the gradient may overwrite the logits
                row_grad<T, NT, ENT_GRAD>(row, x, row_out<T>(L, b, t), L.V, L.c2,
                                          grad_seed(a.m, a.s, st.h, o.g_lp, o.g_h, tok, L.V, L.c));
            }
        } else if (GRAD) {
            row_fill<T, NT>(row_out<T>(L, b, t), L.V, 0.0f);
        }
        if (threadIdx.x == 0) {
            if (p.logprobs) p.logprobs[r] = (float)lp;
            if (p.entropy) p.entropy[r] = st.h;
            if (!GRAD && p.stats) {
                p.stats[r] = st;
                p.g_lp[r] = o.g_lp;
                p.g_h[r] = o.g_h;
            }
        }
    }
    if (threadIdx.x == 0) p.part[blockIdx.x] = total;
}

// ------------------------------------------------------------------------------------------ preference loss
// One workgroup a pair: both sequences' sums in fp64, the pair's loss and dL/dlogp of all of a sequence's tokens.
__global__ __launch_bounds__(256) void pair_kernel(const double* __restrict__ lp, const uint8_t* __restrict__ mask,
                                                   const float* __restrict__ ref, int64_t n_pairs, int64_t n_tok,
                                                   double beta, double smooth, double scale, float* rewards,
                                                   float* seeds, double* part) {
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
            part[q] = scale * ((1.0 - smooth) * neg + (smooth != 0.0 ? smooth * pos : 0.0)) / (double)n_pairs;   // pos may be inf
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
};

struct Teacher {              // one row's entries, in LDS
    int index[PPO_MAX_TEACHER_TOP];     // -1: padding
    float q[PPO_MAX_TEACHER_TOP];       // teacher's probability of the entry
    float all[PPO_MAX_TEACHER_TOP];     // the same summed over the entries of this index
    float u[PPO_MAX_TEACHER_TOP];       // the student's logit there
    float entropy, loss;                // sum q ln q; the row's loss
    int bad, some;                      // a token beyond the vocabulary; an entry that is not padding
};

// Reads the row's entries and makes them probabilities; two barriers at least lie before any of it is used.
template <typename T, int NT>
__device__ __forceinline__ void teacher_load(const TeacherArgs& p, const Logits& L, int64_t r, const T* x, Teacher& s) {
    __syncthreads();          // the previous row's entries have been used
    if (threadIdx.x == 0) s.bad = s.some = 0;
    __syncthreads();
    for (int k = threadIdx.x; k < p.K; k += NT) {
        const int64_t i = int_at(p.index, p.i64, r * p.K + k);
        const bool there = i >= 0 && i < L.V;
        if (i >= L.V) s.bad = 1;
        if (there) s.some = 1;
        s.index[k] = there ? (int)i : -1;
        s.q[k] = there ? float_at(p.logit, p.dtype, r * p.K + k) : 0.0f;
        s.u[k] = there ? wide(x[i]) : 0.0f;
    }
    __syncthreads();
    if (threadIdx.x < 64) {   // softmax over at most PPO_MAX_TEACHER_TOP entries: one wave
        float mx = -__FLT_MAX__, total = 0.0f;
        for (int k = threadIdx.x; k < p.K; k += 64)
            if (s.index[k] >= 0) mx = fmaxf(mx, s.q[k]);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
        for (int k = threadIdx.x; k < p.K; k += 64) {
            const float e = s.index[k] >= 0 ? expf((s.q[k] - mx) * L.c) : 0.0f;
            s.all[k] = (s.q[k] - mx) * L.c;
            s.q[k] = e;
            total += e;
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) total += __shfl_xor(total, off);
        float ent = 0.0f;     // sum q ln q
        const float lt = (float)ln_of(total);
        for (int k = threadIdx.x; k < p.K; k += 64) {
            if (s.index[k] < 0) continue;
            const float q = s.q[k] / total;
            s.q[k] = q;
            if (q != 0.0f) ent = fmaf(q, s.all[k] - lt, ent);
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) ent += __shfl_xor(ent, off);
        if (threadIdx.x == 0) s.entropy = ent;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < p.K; k += NT) {
        float all = 0.0f;
        for (int j = 0; j < p.K; ++j) all += s.index[j] == s.index[k] ? s.q[j] : 0.0f;
        s.all[k] = all;
    }
}

// sum q (ln q - ln p), the same bits on every thread
__device__ __forceinline__ float teacher_loss(const TeacherArgs& p, Teacher& s, float m, float c, double ln_s) {
    __syncthreads();
    if (threadIdx.x < 64) {
        double cross = 0.0;
        for (int k = threadIdx.x; k < p.K; k += 64)
            if (s.index[k] >= 0 && s.q[k] != 0.0f)
                cross += (double)s.q[k] * (((double)s.u[k] - (double)m) * (double)c - ln_s);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) cross += __shfl_xor(cross, off);
        if (threadIdx.x == 0) s.loss = s.bad ? __builtin_nanf("") : (float)((double)s.entropy - cross);
    }
    __syncthreads();
    return s.loss;
}

// dL/dx_i = g (p_i - sum of the teacher's q at i): the bulk first, the K places after a barrier.  A teacher that gave
// nothing teaches nothing.
__device__ __forceinline__ RowGrad teacher_seed(const Teacher& s, float m, float sum, float g) {
    return {m, s.bad ? __builtin_nanf("") : s.some ? g / sum : 0.0f, 0.0f, 0.0f, -1};
}

template <typename T, int NT>
__device__ __forceinline__ void teacher_places(const TeacherArgs& p, const Teacher& s, T* out, const Logits& L,
                                               const RowGrad& rg, float g) {
    __syncthreads();          // the bulk is written
    if (s.bad) return;
    for (int k = threadIdx.x; k < p.K; k += NT)
        if (s.index[k] >= 0) out[s.index[k]] = (T)(grad_of<false>(rg, s.u[k], L.c2) - g * s.all[k]);
}

template <typename T, int NT, bool GRAD>
__global__ __launch_bounds__(NT, 4) void distill_kernel(Logits L, TeacherArgs p) {
    __shared__ Acc lds[NT / 64];
    __shared__ Teacher teach;
    const float temp = 1.0f / L.c;
    double total = 0.0;
    for (int64_t r = blockIdx.x; r < L.n; r += gridDim.x) {
        const int64_t b = r / L.n_tok, t = r - b * L.n_tok;
        RowStats st = {0.0f, 1.0f, 0.0f, 0.0f};
        float loss = 0.0f;
        if (!p.w.mask || p.w.mask[r]) {
            const T* x = row_in<T>(L, b, t);
            Row<T, NT> row;
            row.load(x, L.V);
            teacher_load<T, NT>(p, L, r, x, teach);
            const Acc a = row_stats<T, NT, false>(row, x, L.V, L.c2, lds);
            loss = temp * temp * teacher_loss(p, teach, a.m, L.c, ln_of(a.s));
            st.m = a.m;
            st.s = a.s;
            st.w = row_weight(p.w, b, L.n_tok);
            total += (double)st.w * (double)loss;
            if (GRAD) {
                T* out = row_out<T>(L, b, t);
                const RowGrad g = teacher_seed(teach, a.m, a.s, st.w * temp);
                row_grad<T, NT, false>(row, x, out, L.V, L.c2, g);
                teacher_places<T, NT>(p, teach, out, L, g, st.w * temp);
            }
        } else if (GRAD) {
            row_fill<T, NT>(row_out<T>(L, b, t), L.V, 0.0f);
        }
        if (threadIdx.x == 0) {
            if (p.losses) p.losses[r] = loss;
            if (!GRAD && p.stats) p.stats[r] = st;
        }
    }
    if (threadIdx.x == 0) p.part[blockIdx.x] = total;
}

template <typename T, int NT>
__global__ __launch_bounds__(NT, 4) void distill_backward_kernel(Logits L, TeacherArgs p) {
    __shared__ Teacher teach;
    const float f = (p.factor ? *p.factor : 1.0f) / L.c;
    for (int64_t r = blockIdx.x; r < L.n; r += gridDim.x) {
        const int64_t b = r / L.n_tok, t = r - b * L.n_tok;
        T* out = row_out<T>(L, b, t);
        if (p.w.mask && !p.w.mask[r]) {
            row_fill<T, NT>(out, L.V, 0.0f);
            continue;
        }
        const T* x = row_in<T>(L, b, t);
        const RowStats st = p.stats[r];
        teacher_load<T, NT>(p, L, r, x, teach);
        __syncthreads();
        const RowGrad g = teacher_seed(teach, st.m, st.s, f * st.w);
        row_map<T, NT, false>(x, out, L.V, L.c2, g);
        teacher_places<T, NT>(p, teach, out, L, g, f * st.w);
    }
}

// ------------------------------------------------------------------------------------------ host side
#define ALIGN256(n) (((size_t)(n) + 255) & ~(size_t)255)

struct Workspace {            // one call's scratch
    double* part;             // MAX_GRID partial losses, or one for each pair
    int *totals, *seq_len;
    double* lp64;             // the pairs' log-probabilities
    float* seeds;             // and their gradients
    RowStats* stats;
    size_t bytes;
};

static Workspace carve(void* base, int64_t n_seq, int64_t n_tok) {
    Workspace w;
    char* p = (char*)base;
    auto take = [&](size_t bytes) { char* q = p; p += ALIGN256(bytes); return q; };
    w.part = (double*)take(8 * (size_t)(n_seq > MAX_GRID ? n_seq : MAX_GRID));
    w.totals = (int*)take(8);
    w.seq_len = (int*)take(4 * (size_t)n_seq);
    w.lp64 = (double*)take(8 * (size_t)(n_seq * n_tok));
    w.seeds = (float*)take(4 * (size_t)n_seq);
    w.stats = (RowStats*)take(sizeof(RowStats) * (size_t)(n_seq * n_tok));
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
    if (!(x->inv_temperature > 0.0f) || !(x->inv_temperature < 1e30f)) return PPO_E_BADARG;
    if (x->vocab > PPO_MAX_VOCAB || (x->n_tok > 0 && x->n_seq > PPO_MAX_TOKENS / x->n_tok) || x->n_seq > PPO_MAX_TOKENS)
        return PPO_E_UNSUPPORTED;
    const int64_t n = x->n_seq * x->n_tok;
    if (n == 0) return 0;
    const uintptr_t size = x->dtype == PPO_F32 ? 4 : 2;
    if (!x->data || (uintptr_t)x->data % size || (uintptr_t)grad % size) return PPO_E_BADARG;
    if (grad) {               // rows of the gradient must not overlap
        const int64_t s = x->grad_seq_stride, t = x->grad_tok_stride;
        if ((x->n_tok > 1 && t < x->vocab) || (x->n_seq > 1 && s < (x->n_tok - 1) * t + x->vocab)) return PPO_E_BADARG;
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
    L.V = (int)x->vocab;
    L.c = x->inv_temperature;
    L.c2 = x->inv_temperature * LOG2E_F;
    return L;
}

static int grid_of(int64_t n) { return (int)(n < MAX_GRID ? n : MAX_GRID); }

#define BY_TYPE(dtype, T, ...)                                                     \
    if ((dtype) == PPO_F32) { using T = float; __VA_ARGS__; }                      \
    else if ((dtype) == PPO_BF16) { using T = __bf16; __VA_ARGS__; }               \
    else { using T = _Float16; __VA_ARGS__; }

// Threads of a row: as few as hold it (a row is then in flight as a whole, and the more rows a CU has under way, the
// more of one's memory time hides another's arithmetic).
static int threads_of(const Logits& L, int dtype) {
    const int64_t bytes = (int64_t)L.V * (dtype == PPO_F32 ? 4 : 2);
    int nt = 64;
    while (nt < 1024 && (int64_t)nt * HELD * 16 < bytes) nt *= 2;
    return nt;
}

#define BY_THREADS(threads, NT, ...)                                               \
    switch (threads) {                                                             \
        case 64: { constexpr int NT = 64; __VA_ARGS__; break; }                    \
        case 128: { constexpr int NT = 128; __VA_ARGS__; break; }                  \
        case 256: { constexpr int NT = 256; __VA_ARGS__; break; }                  \
        case 512: { constexpr int NT = 512; __VA_ARGS__; break; }                  \
        default: { constexpr int NT = 1024; __VA_ARGS__; break; }                  \
    }
#define BY_TYPE_AND_THREADS(dtype, threads, T, NT, ...) BY_TYPE(dtype, T, BY_THREADS(threads, NT, __VA_ARGS__))

// Counted rows of each sequence and of all, where a weight needs them.
static void count_rows(const uint8_t* mask, int reduction, const ppo_token_logits* x, const Workspace& w, hipStream_t st) {
    if (!mask || reduction == RED_SUM || x->n_seq * x->n_tok == 0) return;
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
    *o = {mask, w.seq_len, w.totals, reduction, scale, x->n_seq};
    return 0;
}

extern "C" int ppo_token_logprobs(const ppo_token_logits* x, const void* tokens, int tokens_are_i64,
                                  const uint8_t* mask, float* logprobs, float* entropy, float* row_stats, void* stream) {
    const int e = check_logits(x, nullptr);
    if (e) return e;
    const Logits L = logits_of(x, nullptr);
    if (L.n == 0) return 0;
    if (!tokens || !logprobs) return PPO_E_BADARG;
    BY_TYPE_AND_THREADS(x->dtype, threads_of(L, x->dtype), T, NT, {
        if (entropy) logprobs_kernel<T, NT, true><<<grid_of(L.n), NT, 0, (hipStream_t)stream>>>(
            L, tokens, tokens_are_i64, mask, logprobs, nullptr, entropy, (RowStats*)row_stats);
        else logprobs_kernel<T, NT, false><<<grid_of(L.n), NT, 0, (hipStream_t)stream>>>(
            L, tokens, tokens_are_i64, mask, logprobs, nullptr, nullptr, (RowStats*)row_stats);
    })
    return (int)hipGetLastError();
}

static int launch_backward(const Logits& L, int dtype, const void* tokens, int i64, const uint8_t* mask,
                           const RowStats* stats, const Incoming& in, hipStream_t st) {
    constexpr int NT = 256;
    BY_TYPE(dtype, T, {
        if (in.h) backward_kernel<T, NT, true><<<grid_of(L.n), NT, 0, st>>>(L, tokens, i64, mask, stats, in);
        else backward_kernel<T, NT, false><<<grid_of(L.n), NT, 0, st>>>(L, tokens, i64, mask, stats, in);
    })
    return (int)hipGetLastError();
}

extern "C" int ppo_token_logprobs_backward(const ppo_token_logits* x, const void* tokens, int tokens_are_i64,
                                           const uint8_t* mask, const float* row_stats, const float* grad_logprobs,
                                           int64_t lp_seq_stride, int64_t lp_tok_stride, const float* grad_entropy,
                                           int64_t ent_seq_stride, int64_t ent_tok_stride, const float* grad_factor,
                                           void* grad, void* stream) {
    const int e = check_logits(x, grad);
    if (e) return e;
    const Logits L = logits_of(x, grad);
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
    const Logits L = logits_of(x, grad);
    PolicyArgs p;
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
        count_rows(mask, terms->reduction, x, w, st);
        BY_TYPE_AND_THREADS(x->dtype, threads_of(L, x->dtype), T, NT, {
            if (!grad) policy_kernel<T, NT, false, false><<<grid_of(L.n), NT, 0, st>>>(L, p);
            else if (p.ent != 0.0f) policy_kernel<T, NT, true, true><<<grid_of(L.n), NT, 0, st>>>(L, p);
            else policy_kernel<T, NT, true, false><<<grid_of(L.n), NT, 0, st>>>(L, p);
        })
    }
    total_kernel<<<1, 1024, 0, st>>>(w.part, grid_of(L.n), loss);
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
    const Logits L = logits_of(x, grad);
    if (L.n > 0 && !tokens) return PPO_E_BADARG;
    const int64_t pairs = x->n_seq / 2;
    RowStats* stats = row_stats ? (RowStats*)row_stats : w.stats;
    float* sd = seeds ? seeds : w.seeds;
    if (L.n > 0) {
        BY_TYPE_AND_THREADS(x->dtype, threads_of(L, x->dtype), T, NT, (logprobs_kernel<T, NT, false><<<grid_of(L.n), NT, 0, st>>>(
            L, tokens, tokens_are_i64, mask, nullptr, w.lp64, nullptr, stats)))
    }
    pair_kernel<<<grid_of(pairs), 256, 0, st>>>(w.lp64, mask, ref_logprobs, pairs, x->n_tok, beta, label_smoothing, scale,
                                                rewards, sd, w.part);
    total_kernel<<<1, 1024, 0, st>>>(w.part, (int)pairs, loss);
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
    e = weights_of(&p.w, mask, reduction, scale, x, w);
    if (e) return e;
    const Logits L = logits_of(x, grad);
    p.losses = token_losses;
    p.stats = (RowStats*)row_stats;
    p.part = w.part;
    if (L.n > 0) {
        count_rows(mask, reduction, x, w, st);
        BY_TYPE_AND_THREADS(x->dtype, threads_of(L, x->dtype), T, NT, {
            if (grad) distill_kernel<T, NT, true><<<grid_of(L.n), NT, 0, st>>>(L, p);
            else distill_kernel<T, NT, false><<<grid_of(L.n), NT, 0, st>>>(L, p);
        })
    }
    total_kernel<<<1, 1024, 0, st>>>(w.part, grid_of(L.n), loss);
    return (int)hipGetLastError();
}

extern "C" int ppo_distillation_backward(const ppo_token_logits* x, const void* teacher_tokens, int tokens_are_i64,
                                         const void* teacher_logits, int teacher_dtype, int top, const uint8_t* mask,
                                         const float* row_stats, const float* grad_factor, void* grad, void* stream) {
    int e = check_logits(x, grad);
    TeacherArgs p;
    if (!e) e = teacher_of(&p, x, teacher_tokens, tokens_are_i64, teacher_logits, teacher_dtype, top);
    if (e) return e;
    const Logits L = logits_of(x, grad);
    if (L.n == 0) return 0;
    if (!row_stats || !grad) return PPO_E_BADARG;
    p.w.mask = mask;
    p.stats = (RowStats*)row_stats;
    p.factor = grad_factor;
    constexpr int NT = 256;
    BY_TYPE(x->dtype, T, (distill_backward_kernel<T, NT><<<grid_of(L.n), NT, 0, (hipStream_t)stream>>>(L, p)))
    return (int)hipGetLastError();
}
