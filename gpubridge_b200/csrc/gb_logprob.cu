// Log-probabilities of sampled tokens over a vocabulary, the losses of fine-tuning that are made
// of them, and their gradient with respect to the logits.
//
//   logprob_r = x_t / T - log sum_j exp(x_j / T)                       (t: the row's target)
//   policy loss:      ratio = exp(logprob - old),  gap = ref - logprob
//                     l_r = -min(ratio A, clip(ratio, 1 - lo, 1 + hi) A) + c (exp(gap) - 1 - gap)
//                     loss = sum w_r l_r / D
//   preference loss:  S_s = sum (or mean) of a sequence's logprobs,  reward_s = beta (S_s - ref_s)
//                     m = reward(chosen) - reward(rejected)
//                     loss = mean over pairs of -(1 - e) log sigmoid(m) - e log sigmoid(-m)
//   gradient:         d x_j = coef_r / T * ([j = t] - p_j),  p_j = exp(x_j / T) / sum
//
// Every loss gives each row one coefficient, so the gradient is one more sweep over the row.  The
// policy loss knows a row's coefficient as soon as its sum is there: one launch reads a row,
// and sweeps it again out of L2 to write the gradient.  The preference loss needs whole sequences
// first: forward reads the logits, backward reads them again and writes.
//
// A block owns a row.  A row may begin at any address: a vector that reaches over the row's end
// is handled value by value, and a gradient's row lies across the vectors as the logits' row does.  Rows whose
// target is outside the vocabulary, or whose weight is 0, are not read; their gradient is 0.
// Row sums are in fp32 (a thread adds a few hundred terms in [0, 1], the block joins 512 of them),
// sums over rows in 64 bits and in a fixed order.  Bound by memory.
#include <math_constants.h>
#include "gb_vec.cuh"

namespace {

constexpr int THREADS = 512;
constexpr float LOG2E = 1.4426950408889634f;

// 2^x by the special-function unit (2 ulp; below 2^-126 it gives 0, which no sum here resolves).
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T> struct Pack16 {                 // 16 bytes
    static constexpr int N = 16 / (int)sizeof(T);
    uint4 q;
    __device__ __forceinline__ void load(const T* p) { q = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void get(float (&v)[N]) const {
        if constexpr (sizeof(T) == 4) {
            v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y);
            v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
        } else {
            Raw8<T> raw;
            raw.q = q;
            raw.get(v);
        }
    }
    static __device__ __forceinline__ void store(T* p, const float (&v)[N]) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        else gb_store8(p, v);
    }
};

// Rows of logits: row r is row r % inner of batch entry r / inner.
struct Rows {
    const void* x;
    long long batch_stride, row_stride, inner, rows;
    int vocab, ld;                       // columns that count, columns there are
    __device__ __forceinline__ long long offset(long long r) const {
        const long long b = r / inner;
        return b * batch_stride + (r - b * inner) * row_stride;
    }
};

// A row in vectors: vector i holds the columns i * N - skew ...
template <typename T>
struct Row {
    static constexpr int N = Pack16<T>::N;
    const T* base;                       // 16-byte aligned, at or before the row's first value
    int skew, vocab, full_lo, full_hi, vectors;   // [full_lo, full_hi): vectors wholly in the vocabulary
    __device__ Row(const T* x, int vocab_) : vocab(vocab_) {
        skew = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
        base = x - skew;
        vectors = (vocab + skew + N - 1) / N;
        full_lo = skew ? 1 : 0;
        full_hi = (vocab + skew) / N;
    }
    __device__ __forceinline__ bool full(int i) const { return i >= full_lo && i < full_hi; }
    // any vector; columns outside the vocabulary read as -inf
    __device__ __forceinline__ void load(int i, float (&v)[N]) const {
        if (full(i)) {
            Pack16<T> p;
            p.load(base + (long long)i * N);
            p.get(v);
        } else {
            #pragma unroll
            for (int j = 0; j < N; ++j) {
                const int col = i * N - skew + j;
                v[j] = (col >= 0 && col < vocab) ? gb_up(base[(long long)i * N + j]) : -CUDART_INF_F;
            }
        }
    }
};

// Running maximum m and sum s of exp2((x - m) * k).  One vector at a time: its maximum decides
// whether the sum is rescaled, rare after the first few.
template <int N>
__device__ __forceinline__ void take(const float (&v)[N], float k, float& m, float& s) {
    float top = v[0];
    #pragma unroll
    for (int j = 1; j < N; ++j) top = fmaxf(top, v[j]);
    if (top > m) { s *= fast_exp2((m - top) * k); m = top; }
    if (m == -CUDART_INF_F) {                        // nothing finite yet; a NaN must not get lost
        #pragma unroll
        for (int j = 0; j < N; ++j) if (v[j] != v[j]) s = v[j];
        return;
    }
    #pragma unroll
    for (int j = 0; j < N; ++j) s += fast_exp2((v[j] - m) * k);
}

__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2, float k) {
    const float top = fmaxf(m, m2);
    if (top == -CUDART_INF_F) { s += s2; return; }
    s = s * fast_exp2((m - top) * k) + s2 * fast_exp2((m2 - top) * k);
    m = top;
}

// (maximum, sum) of the row, in every thread.
template <typename T>
__device__ float2 row_stats(const Row<T>& row, float k) {
    constexpr int N = Row<T>::N;
    float m = -CUDART_INF_F, s = 0.0f;
    int i = threadIdx.x;
    for (; i + THREADS < row.full_hi; i += 2 * THREADS) {
        if (i >= row.full_lo) {
            Pack16<T> a, b;
            a.load(row.base + (long long)i * N);
            b.load(row.base + (long long)(i + THREADS) * N);
            float v[N];
            a.get(v);
            take<N>(v, k, m, s);
            b.get(v);
            take<N>(v, k, m, s);
        } else {
            float v[N];
            row.load(i, v);
            take<N>(v, k, m, s);
            row.load(i + THREADS, v);
            take<N>(v, k, m, s);
        }
    }
    for (; i < row.vectors; i += THREADS) {
        float v[N];
        row.load(i, v);
        take<N>(v, k, m, s);
    }
    __shared__ float2 part[THREADS / 32];
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
        merge(m, s, m2, s2, k);
    }
    __syncthreads();                                 // the last row's results may still be read
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = make_float2(m, s);
    __syncthreads();
    m = part[0].x; s = part[0].y;
    #pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) merge(m, s, part[w].x, part[w].y, k);
    return make_float2(m, s);
}

// The gradient of a row whose log-probability has the gradient `coef`: zeros from vocab to ld.
// `out` lies in its vectors as the row does.
template <typename T>
__device__ void write_grad(const Row<T>& row, T* out, int ld, int target, float coef, float2 stats, float k,
                           float inv_temperature) {
    constexpr int N = Row<T>::N;
    const float scale = -coef * inv_temperature / stats.y, hit = coef * inv_temperature;
    T* base = out - row.skew;
    const int vectors = (ld + row.skew + N - 1) / N, full_hi = (ld + row.skew) / N;
    const int at = target + row.skew;
    for (int i = threadIdx.x; i < vectors; i += THREADS) {
        float v[N];
        row.load(i, v);
        #pragma unroll
        for (int j = 0; j < N; ++j) {
            v[j] = fast_exp2((v[j] - stats.x) * k) * scale;
            if (!row.full(i) && i * N - row.skew + j >= row.vocab) v[j] = 0.0f;
        }
        if (i == at / N) {
            #pragma unroll
            for (int j = 0; j < N; ++j) if (j == at % N) v[j] += hit;
        }
        if (i >= row.full_lo && i < full_hi) Pack16<T>::store(base + (long long)i * N, v);
        else {
            #pragma unroll
            for (int j = 0; j < N; ++j) {
                const int col = i * N - row.skew + j;
                if (col >= 0 && col < ld) base[(long long)i * N + j] = gb_down<T>(v[j]);
            }
        }
    }
}

template <typename T>
__device__ void write_zeros(const Row<T>& row, T* out, int ld) {
    constexpr int N = Row<T>::N;
    T* base = out - row.skew;
    const int vectors = (ld + row.skew + N - 1) / N, full_hi = (ld + row.skew) / N;
    const float zero[N] = {};
    for (int i = threadIdx.x; i < vectors; i += THREADS) {
        if (i >= row.full_lo && i < full_hi) Pack16<T>::store(base + (long long)i * N, zero);
        else {
            #pragma unroll
            for (int j = 0; j < N; ++j) {
                const int col = i * N - row.skew + j;
                if (col >= 0 && col < ld) base[(long long)i * N + j] = gb_down<T>(0.0f);
            }
        }
    }
}

// Sum over the block in 64 bits, in a fixed order, in every thread.
__device__ double block_sum(double v) {
    __shared__ double part[THREADS / 32];
    v = gb_warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    double total = part[0];
    for (int w = 1; w < THREADS / 32; ++w) total += part[w];
    return total;
}

struct ForwardArgs {
    Rows rows;
    const long long* targets;
    float inv_temperature;
    float* logprobs;                     // [rows]
    float2* stats;                       // [rows] maximum and sum, or null
    // the policy loss
    const float *old, *advantages, *ref, *weights, *denominator;
    float clip_low, clip_high, kl_coef;
    float* coef;                         // [rows] gradient of the loss by each log-probability
    float* terms;                        // [3][rows] weighted loss, kl, clipped
    float* inv_denominator;
    void* grad;                          // null: none is written
};

enum { LOGPROBS = 0, POLICY = 1 };

template <typename T, int MODE>
__global__ void __launch_bounds__(THREADS) forward_kernel(const ForwardArgs a) {
    __shared__ float s_coef;
    float inv = 1.0f;
    if (MODE == POLICY) {
        double d;
        if (a.denominator) d = *a.denominator;
        else {                           // every block adds the weights for itself: no second launch
            d = 0.0;
            for (long long r = threadIdx.x; r < a.rows.rows; r += THREADS) {
                const long long t = a.targets[r];
                if (t >= 0 && t < a.rows.vocab) d += a.weights ? (double)a.weights[r] : 1.0;
            }
            d = block_sum(d);
        }
        inv = d == 0.0 ? 0.0f : (float)(1.0 / d);    // no token counts: loss and gradient are 0
        if (blockIdx.x == 0 && threadIdx.x == 0) *a.inv_denominator = inv;
    }
    const float k = LOG2E * a.inv_temperature;
    for (long long r = blockIdx.x; r < a.rows.rows; r += gridDim.x) {
        const long long at = a.rows.offset(r);
        const T* x = static_cast<const T*>(a.rows.x) + at;
        const Row<T> row(x, a.rows.vocab);
        const long long target = a.targets[r];
        const float weight = (MODE == POLICY && a.weights) ? a.weights[r] : 1.0f;
        const bool counted = target >= 0 && target < a.rows.vocab && weight != 0.0f;
        T* out = a.grad ? static_cast<T*>(a.grad) + r * a.rows.ld : nullptr;
        if (!counted) {
            if (threadIdx.x == 0) {
                a.logprobs[r] = 0.0f;
                if (a.stats) a.stats[r] = make_float2(0.0f, 1.0f);
                if (MODE == POLICY) {
                    a.coef[r] = 0.0f;
                    for (int q = 0; q < 3; ++q) a.terms[q * a.rows.rows + r] = 0.0f;
                }
            }
            if (out) write_zeros(row, out, a.rows.ld);
            continue;
        }
        const float2 stats = row_stats(row, k);
        if (threadIdx.x == 0) {
            const float logprob = (gb_up(x[target]) - stats.x) * a.inv_temperature - logf(stats.y);
            a.logprobs[r] = logprob;
            if (a.stats) a.stats[r] = stats;
            if (MODE == POLICY) {
                const float adv = a.advantages[r];
                const float ratio = expf(logprob - a.old[r]);
                const float low = 1.0f - a.clip_low, high = 1.0f + a.clip_high;
                const bool outside = (adv > 0.0f && ratio > high) || (adv < 0.0f && ratio < low);
                float loss = -fminf(ratio * adv, fminf(fmaxf(ratio, low), high) * adv);
                if (ratio != ratio || adv != adv) loss = ratio * adv;        // a NaN stays one
                float d = outside ? 0.0f : -adv * ratio;
                float kl = 0.0f;
                if (a.ref) {
                    const float gap = a.ref[r] - logprob, e = expm1f(gap);
                    kl = e - gap;
                    loss += a.kl_coef * kl;
                    d -= a.kl_coef * e;
                }
                a.terms[r] = weight * loss;
                a.terms[a.rows.rows + r] = weight * kl;
                a.terms[2 * a.rows.rows + r] = outside ? weight : 0.0f;
                s_coef = weight * inv * d;
                a.coef[r] = s_coef;
            }
        }
        if (MODE == POLICY && out) {
            __syncthreads();
            const float coef = s_coef;
            if (coef == 0.0f) write_zeros(row, out, a.rows.ld);
            else write_grad(row, out, a.rows.ld, (int)target, coef, stats, k, a.inv_temperature);
        }
    }
}

// The three sums of terms times the reciprocal denominator.
__global__ void __launch_bounds__(THREADS) policy_finish_kernel(const float* __restrict__ terms, long long rows,
                                                                const float* inv, float* loss, float* kl,
                                                                float* clipped) {
    for (int q = 0; q < 3; ++q) {
        double acc = 0.0;
        for (long long r = threadIdx.x; r < rows; r += THREADS) acc += terms[q * rows + r];
        acc = block_sum(acc);
        if (threadIdx.x == 0) *(q == 0 ? loss : q == 1 ? kl : clipped) = (float)(acc * (double)*inv);
    }
}

struct GradArgs {
    Rows rows;
    const long long* targets;
    const float2* stats;
    const float* coef;                   // [rows]
    const float* upstream;               // one value that multiplies every coefficient, or null
    float inv_temperature;
    void* grad;
};

template <typename T>
__global__ void __launch_bounds__(THREADS) grad_kernel(const GradArgs a) {
    const float up = a.upstream ? *a.upstream : 1.0f;
    const float k = LOG2E * a.inv_temperature;
    for (long long r = blockIdx.x; r < a.rows.rows; r += gridDim.x) {
        const long long at = a.rows.offset(r);
        const Row<T> row(static_cast<const T*>(a.rows.x) + at, a.rows.vocab);
        T* out = static_cast<T*>(a.grad) + r * a.rows.ld;
        const long long target = a.targets[r];
        const float own = a.coef[r], coef = own * up;
        if (target < 0 || target >= a.rows.vocab || own == 0.0f || coef == 0.0f) write_zeros(row, out, a.rows.ld);
        else write_grad(row, out, a.rows.ld, (int)target, coef, a.stats[r], k, a.inv_temperature);
    }
}

struct PreferenceArgs {
    const float* logprobs;               // [rows]
    const long long* targets;
    const long long* offsets;            // [sequences + 1] first row of each, or null: `length` rows each
    long long rows, length;
    int sequences, vocab, average;
    const void* ref;                     // [sequences] float or double
    int ref_double;
    double beta, smoothing;
    double* sums;                        // [sequences]
    float* seq_coef;                     // [sequences]
    float *loss, *rewards, *seq_logprobs, *coef;
};

// One block: the log-probabilities are a few bytes a row next to the logits' hundred thousand.
__global__ void __launch_bounds__(THREADS) preference_kernel(const PreferenceArgs a) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = THREADS / 32;
    auto begin = [&](int s) {
        long long v = a.offsets ? a.offsets[s] : s * a.length;
        return v < 0 ? 0LL : (v > a.rows ? a.rows : v);      // whatever the offsets hold, rows are in range
    };
    for (int s = warp; s < a.sequences; s += warps) {
        const long long lo = begin(s), hi = begin(s + 1);
        double sum = 0.0, tokens = 0.0;
        for (long long r = lo + lane; r < hi; r += 32) {
            sum += a.logprobs[r];
            tokens += (a.targets[r] >= 0 && a.targets[r] < a.vocab) ? 1.0 : 0.0;
        }
        sum = gb_warp_sum(sum);
        tokens = gb_warp_sum(tokens);
        if (lane == 0) {
            const double share = a.average ? 1.0 / (tokens > 1.0 ? tokens : 1.0) : 1.0;
            a.sums[s] = sum * share;
            a.seq_coef[s] = (float)share;
            const double ref = a.ref_double ? static_cast<const double*>(a.ref)[s] : static_cast<const float*>(a.ref)[s];
            a.seq_logprobs[s] = (float)(sum * share);
            a.rewards[s] = (float)(a.beta * (sum * share - ref));
        }
    }
    __syncthreads();
    const int pairs = a.sequences / 2;
    double loss = 0.0;
    for (int p = threadIdx.x; p < pairs; p += THREADS) {
        auto reward = [&](int s) {
            const double ref = a.ref_double ? static_cast<const double*>(a.ref)[s] : static_cast<const float*>(a.ref)[s];
            return a.beta * (a.sums[s] - ref);
        };
        const double m = reward(p) - reward(p + pairs);
        // -log sigmoid(m) = log(1 + exp(-|m|)) + max(-m, 0)
        const double soft = log1p(exp(-fabs(m)));
        loss += (1.0 - a.smoothing) * (soft + fmax(-m, 0.0)) + a.smoothing * (soft + fmax(m, 0.0));
        if (m != m) loss = m;
        const double sigmoid = m >= 0.0 ? 1.0 / (1.0 + exp(-m)) : exp(m) / (1.0 + exp(m));
        const double d = (sigmoid - (1.0 - a.smoothing)) * a.beta / pairs;
        a.seq_coef[p] = (float)(d * (double)a.seq_coef[p]);
        a.seq_coef[p + pairs] = (float)(-d * (double)a.seq_coef[p + pairs]);
    }
    loss = block_sum(loss);                          // its barriers also publish seq_coef
    if (threadIdx.x == 0) *a.loss = (float)(loss / pairs);
    for (long long r = threadIdx.x; r < begin(0); r += THREADS) a.coef[r] = 0.0f;
    for (long long r = begin(a.sequences) + threadIdx.x; r < a.rows; r += THREADS) a.coef[r] = 0.0f;
    for (int s = warp; s < a.sequences; s += warps) {
        const float c = a.seq_coef[s];
        for (long long r = begin(s) + lane; r < begin(s + 1); r += 32) a.coef[r] = c;
    }
}

int grid_for(long long rows) { return (int)(rows < 148 * 4 ? rows : 148 * 4); }

bool bad(const Rows& r) {
    return r.rows <= 0 || r.inner <= 0 || r.vocab <= 0 || r.ld < r.vocab || r.ld > 0x7fffff00;
}

}  // namespace

// dtype: codes of gb_vec.cuh.  logits: row r begins batch_stride * (r / inner) + row_stride *
// (r % inner) values behind `logits`; vocab of its ld columns count.  targets: int64, -1 or anything
// else outside [0, vocab) for a row that does not count.  grad, where it is given, is [rows, ld]
// without gaps, and each of its rows is as far from a 16-byte boundary as the logits' row.
extern "C" int gb_token_logprobs(int dtype, const void* logits, long long batch_stride, long long row_stride,
                                 long long inner, long long rows, int vocab, int ld, const long long* targets,
                                 float temperature, float* logprobs, float* stats, cudaStream_t stream) {
    ForwardArgs a = {};
    a.rows = Rows{logits, batch_stride, row_stride, inner, rows, vocab, ld};
    if (bad(a.rows)) return (int)cudaErrorInvalidValue;
    a.targets = targets; a.inv_temperature = 1.0f / temperature; a.logprobs = logprobs;
    a.stats = reinterpret_cast<float2*>(stats);
    const int grid = grid_for(rows);
    if (dtype == GB_F32) forward_kernel<float, LOGPROBS><<<grid, THREADS, 0, stream>>>(a);
    else if (dtype == GB_BF16) forward_kernel<__nv_bfloat16, LOGPROBS><<<grid, THREADS, 0, stream>>>(a);
    else if (dtype == GB_F16) forward_kernel<__half, LOGPROBS><<<grid, THREADS, 0, stream>>>(a);
    else return (int)cudaErrorInvalidValue;
    return (int)cudaGetLastError();
}

// scratch: 3 * rows + 1 floats.  loss, kl, clipped (share): one float each.  ref, weights and denominator may be
// null; grad null: backward is gb_logprob_grad with `coef` and `stats` (null where grad is given).
extern "C" int gb_policy_loss(int dtype, const void* logits, long long batch_stride, long long row_stride,
                              long long inner, long long rows, int vocab, int ld, const long long* targets,
                              float temperature, const float* old, const float* advantages, const float* ref,
                              const float* weights, const float* denominator, float clip_low, float clip_high,
                              float kl_coef, float* logprobs, float* stats, float* coef, float* scratch,
                              float* loss, float* kl, float* clipped, void* grad, cudaStream_t stream) {
    ForwardArgs a = {};
    a.rows = Rows{logits, batch_stride, row_stride, inner, rows, vocab, ld};
    if (bad(a.rows)) return (int)cudaErrorInvalidValue;
    a.targets = targets; a.inv_temperature = 1.0f / temperature; a.logprobs = logprobs;
    a.stats = reinterpret_cast<float2*>(stats);
    a.old = old; a.advantages = advantages; a.ref = ref; a.weights = weights; a.denominator = denominator;
    a.clip_low = clip_low; a.clip_high = clip_high; a.kl_coef = kl_coef;
    a.coef = coef; a.terms = scratch; a.inv_denominator = scratch + 3 * rows; a.grad = grad;
    const int grid = grid_for(rows);
    if (dtype == GB_F32) forward_kernel<float, POLICY><<<grid, THREADS, 0, stream>>>(a);
    else if (dtype == GB_BF16) forward_kernel<__nv_bfloat16, POLICY><<<grid, THREADS, 0, stream>>>(a);
    else if (dtype == GB_F16) forward_kernel<__half, POLICY><<<grid, THREADS, 0, stream>>>(a);
    else return (int)cudaErrorInvalidValue;
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return (int)err;
    policy_finish_kernel<<<1, THREADS, 0, stream>>>(scratch, rows, scratch + 3 * rows, loss, kl, clipped);
    return (int)cudaGetLastError();
}

extern "C" int gb_logprob_grad(int dtype, const void* logits, long long batch_stride, long long row_stride,
                               long long inner, long long rows, int vocab, int ld, const long long* targets,
                               float temperature, const float* stats, const float* coef, const float* upstream,
                               void* grad, cudaStream_t stream) {
    GradArgs a = {};
    a.rows = Rows{logits, batch_stride, row_stride, inner, rows, vocab, ld};
    if (bad(a.rows)) return (int)cudaErrorInvalidValue;
    a.targets = targets; a.stats = reinterpret_cast<const float2*>(stats); a.coef = coef; a.upstream = upstream;
    a.inv_temperature = 1.0f / temperature; a.grad = grad;
    const int grid = grid_for(rows);
    if (dtype == GB_F32) grad_kernel<float><<<grid, THREADS, 0, stream>>>(a);
    else if (dtype == GB_BF16) grad_kernel<__nv_bfloat16><<<grid, THREADS, 0, stream>>>(a);
    else if (dtype == GB_F16) grad_kernel<__half><<<grid, THREADS, 0, stream>>>(a);
    else return (int)cudaErrorInvalidValue;
    return (int)cudaGetLastError();
}

// sums: `sequences` doubles of scratch, seq_coef: as many floats.  The first half of the sequences
// was chosen over the second half, pair by pair.
extern "C" int gb_preference_loss(const float* logprobs, const long long* targets, const long long* offsets,
                                  long long rows, long long length, int sequences, int vocab, int average,
                                  const void* ref, int ref_double, double beta, double smoothing, double* sums,
                                  float* seq_coef, float* loss, float* rewards, float* seq_logprobs,
                                  float* coef, cudaStream_t stream) {
    if (sequences < 2 || sequences % 2) return (int)cudaErrorInvalidValue;
    const PreferenceArgs a = {logprobs, targets, offsets, rows, length, sequences, vocab, average, ref, ref_double,
                              beta, smoothing, sums, seq_coef, loss, rewards, seq_logprobs, coef};
    preference_kernel<<<1, THREADS, 0, stream>>>(a);
    return (int)cudaGetLastError();
}
