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
// A block owns a row, or a cluster where there are few.  A row may begin at any address: what lies
// before its first whole vector and behind its last is handled value by value, and a gradient's row
// lies across the vectors as the logits' row does.  Rows whose target is outside the vocabulary, or
// whose weight is 0, are not read; their gradient is 0.  Row sums are in fp32 (a thread adds a few
// hundred terms in [0, 1], the block joins 256 of them), sums over rows in 64 bits and in a fixed
// order.
//
// Bound by memory, but closely followed by the instructions: a value costs one exponential a sweep
// and about four others (packed maxima, packed fused multiply-adds).  One B200, 8192 x 50257 bf16:
// log-probabilities 137 us (6.0 TB/s), a policy step 302 us where reading and writing every counted
// row once would take 239.  Five blocks of 256 threads an SM were better than three of 512 (323 us),
// than six (307 us) and than rows kept in shared memory for the second sweep (376 us): what counts
// is loads under way, and the rows in flight (74 MB) mostly stay in L2 when the gradient is stored
// past it (344 us without that).  A preference step of 4096 x 128256 takes 450 us; its two reads and
// one write are 1.84 + 0.79 GB, 407 us.
#include <cooperative_groups.h>
#include <math.h>
#include "gb_vec.cuh"

namespace {

namespace cg = cooperative_groups;

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int BATCH = 4;                             // vectors of 16 bytes that a thread has under way
// 2^x by the special-function unit (2 ulp; below 2^-126 it gives 0, which no sum here resolves).
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^d for a whole d, exactly: 1 above 0, 0 below -126.  1.5 * 2^23 + d has d in its last bits.
__device__ __forceinline__ float whole_exp2(float d) {
    return d < -126.0f ? 0.0f : __int_as_float((__float_as_int(fminf(d, 0.0f) + 12582912.0f) << 23) + 0x3f800000);
}

// The unit's powers are low by 5.0e-8 of themselves on average (4 M values in [-20, -1] on a B200;
// their spread is 5e-8 too, but that averages out).  A sum over a thousand tokens shows it, so the
// logarithm of a row's sum is put right by it.
constexpr double EXP2_LOW = 5.0e-8;

// log2(e) / T in two parts: the rounding of one alone would shift every log-probability the same
// way (by 1e-8 of the logits' spread, which a sum over a thousand tokens shows as well).
struct Base { float k, rest; double inv_temperature; };

// Two values in one instruction (sm_100a's packed fp32); each rounds as the single one does.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)),
          "l"(reinterpret_cast<const unsigned long long&>(c)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 exp2_2(float2 t) { return make_float2(fast_exp2(t.x), fast_exp2(t.y)); }

// 16 bytes of values: their pairs, their maximum, and back.
template <typename T> struct Pack;
template <> struct Pack<float> {
    static constexpr int N = 4;
    static constexpr uint32_t LOW = 0xff800000u;     // -inf in every place
    static __device__ __forceinline__ void pairs(const uint4& q, float2 (&v)[2]) {
        v[0] = make_float2(__uint_as_float(q.x), __uint_as_float(q.y));
        v[1] = make_float2(__uint_as_float(q.z), __uint_as_float(q.w));
    }
    template <int U> static __device__ __forceinline__ float top(const uint4 (&q)[U]) {
        float m = -INFINITY;
        #pragma unroll
        for (int i = 0; i < U; ++i)
            m = fmaxf(fmaxf(m, fmaxf(__uint_as_float(q[i].x), __uint_as_float(q[i].y))),
                      fmaxf(__uint_as_float(q[i].z), __uint_as_float(q[i].w)));
        return m;
    }
    static __device__ __forceinline__ uint4 back(const float2 (&v)[2]) {
        return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
    }
};
template <> struct Pack<__nv_bfloat16> {
    static constexpr int N = 8;
    static constexpr uint32_t LOW = 0xff80ff80u;
    static __device__ __forceinline__ void pairs(const uint4& q, float2 (&v)[4]) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
        #pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
    template <int U> static __device__ __forceinline__ float top(const uint4 (&q)[U]) {
        __nv_bfloat162 m;
        #pragma unroll
        for (int i = 0; i < U; ++i) {
            const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q[i]);
            const __nv_bfloat162 a = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
            m = i ? __hmax2(m, a) : a;
        }
        return fmaxf(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ uint4 back(const float2 (&v)[4]) {
        uint4 q;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
        #pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[i].x, v[i].y);
        return q;
    }
};
template <> struct Pack<__half> {
    static constexpr int N = 8;
    static constexpr uint32_t LOW = 0xfc00fc00u;
    static __device__ __forceinline__ void pairs(const uint4& q, float2 (&v)[4]) {
        const __half2* h = reinterpret_cast<const __half2*>(&q);
        #pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __half22float2(h[i]);
    }
    template <int U> static __device__ __forceinline__ float top(const uint4 (&q)[U]) {
        __half2 m;
        #pragma unroll
        for (int i = 0; i < U; ++i) {
            const __half2* h = reinterpret_cast<const __half2*>(&q[i]);
            const __half2 a = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
            m = i ? __hmax2(m, a) : a;
        }
        return fmaxf(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ uint4 back(const float2 (&v)[4]) {
        uint4 q;
        __half2* h = reinterpret_cast<__half2*>(&q);
        #pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[i].x, v[i].y);
        return q;
    }
};

// Rows of logits: row r is row r % inner of batch entry r / inner.
struct Rows {
    const void* x;
    long long batch_stride, row_stride, inner, rows;
    int vocab, ld;                       // columns that count, columns there are
    __device__ __forceinline__ long long offset(long long r) const {
        if (inner == rows) return r * row_stride;
        const long long b = r / inner;
        return b * batch_stride + (r - b * inner) * row_stride;
    }
};

// A row, or one block's share of its whole vectors.  Vector i holds the columns i * N - skew and
// on; the few columns before the first whole vector and behind the last are the edges.
template <typename T>
struct Row {
    static constexpr int N = Pack<T>::N, P = N / 2;
    const T* x;
    const uint4* base;                   // at or before the row's first value
    int skew, lo, hi;                    // this block's vectors
    int head, tail, vocab;               // edges: columns [0, head) and [tail, vocab)
    __device__ Row(const T* x_, int vocab_, int part, int parts) : x(x_), vocab(vocab_) {
        skew = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
        base = reinterpret_cast<const uint4*>(x - skew);
        int first = skew ? 1 : 0, last = (vocab + skew) / N;
        if (last < first) last = first;
        head = first * N - skew;
        if (head > vocab) head = vocab;
        if (!skew) head = 0;
        tail = last * N - skew;
        if (tail < head) tail = head;
        if (tail > vocab) tail = vocab;
        const int share = (last - first + parts - 1) / parts;
        lo = first + part * share;
        hi = lo + share;
        if (lo > last) lo = last;
        if (hi > last) hi = last;
    }
    __device__ __forceinline__ int edges() const { return head + vocab - tail; }
    __device__ __forceinline__ int edge(int i) const { return i < head ? i : tail + i - head; }
};

// From 2^30 on the product m k is rounded by more than 32, and terms could leave fp32's range: a row
// whose maximum is a mask's -1e9, the type's lowest value, or inf.  Neighbours there are 2^-64 of one
// another, so that a far running maximum may drop its terms once a nearer one is found.
__device__ __forceinline__ bool is_far(float m, float k) { return !(fabsf(m) * k < 1073741824.0f); }

// A row's terms are 2^(x k + c) with c the whole number next to -m k, m the row's maximum: sums of
// different c are joined by powers of two, without a rounding.
__device__ __forceinline__ float offset_for(float m, float k) { return is_far(m, k) ? 0.0f : -rintf(m * k); }

// Running maximum and sum.  The maximum of a batch decides whether the sum is rescaled, which is
// rare after the first few.  While the maximum is far, nothing is summed that counts.
struct Running {
    float m, c, s0;
    float2 s;
    __device__ __forceinline__ Running() : m(-INFINITY), c(0.0f), s0(0.0f), s(both(0.0f)) {}
    __device__ __forceinline__ void raise(float top, float k) {
        if (top > m) {
            const float old = c;
            const bool first = is_far(m, k);
            m = top;
            c = offset_for(m, k);
            if (!first) {
                const float f = whole_exp2(c - old);
                s = mul2(s, both(f));
                s0 *= f;
            }
        }
    }
    __device__ __forceinline__ void add(float x, const Base& b) {
        raise(x, b.k);
        s0 += fast_exp2(fmaf(x, b.rest, fmaf(x, b.k, c)));
    }
};

// Maximum, whole number and sum of a part's terms.  A far part has no terms (its sum is 0, or a NaN).
struct Stats { float m, c, s; };

template <typename F>
__device__ __forceinline__ Stats join(int parts, float k, F part) {
    float m = part(0).m;
    for (int p = 1; p < parts; ++p) m = fmaxf(m, part(p).m);
    Stats all{m, offset_for(m, k), 0.0f};
    for (int p = 0; p < parts; ++p) {
        const Stats one = part(p);
        all.s += one.s * whole_exp2(all.c - one.c);
    }
    return all;
}

template <typename T>
__device__ Stats row_stats(const Row<T>& row, const Base& base, bool with_edges, Stats* part) {
    constexpr int P = Row<T>::P;
    constexpr uint32_t LOW = Pack<T>::LOW;
    Running run;
    const float k = base.k;
    const float2 k2 = both(k), rest2 = both(base.rest);
    // a vector's sum on its own: small terms added to the whole sum one by one would be lost in it
    auto take = [&](const uint4& q) {
        float2 v[P];
        Pack<T>::pairs(q, v);
        const float2 c2 = both(run.c);
        #pragma unroll
        for (int j = 0; j < P; ++j) v[j] = exp2_2(fma2(v[j], rest2, fma2(v[j], k2, c2)));
        #pragma unroll
        for (int j = 1; j < P; ++j) v[0] = add2(v[0], v[j]);
        return v[0];
    };
    int i = row.lo + (int)threadIdx.x;
    for (; i + (BATCH - 1) * THREADS < row.hi; i += BATCH * THREADS) {
        uint4 q[BATCH];
        #pragma unroll
        for (int u = 0; u < BATCH; ++u) q[u] = row.base[i + u * THREADS];
        run.raise(Pack<T>::top(q), k);
        float2 sum = take(q[0]);
        #pragma unroll
        for (int u = 1; u < BATCH; ++u) sum = add2(sum, take(q[u]));
        run.s = add2(run.s, sum);
    }
    if (i < row.hi) {                    // the last batch, with -inf where there is no vector
        uint4 q[BATCH];
        #pragma unroll
        for (int u = 0; u < BATCH; ++u)
            q[u] = i + u * THREADS < row.hi ? row.base[i + u * THREADS] : make_uint4(LOW, LOW, LOW, LOW);
        run.raise(Pack<T>::top(q), k);
        #pragma unroll
        for (int u = 0; u < BATCH; ++u) if (i + u * THREADS < row.hi) run.s = add2(run.s, take(q[u]));
    }
    if (with_edges && (int)threadIdx.x < row.edges()) run.add(gb_up(row.x[row.edge(threadIdx.x)]), base);
    float sum = run.s.x + run.s.y + run.s0, top = run.m;
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float c = offset_for(top, k);
    sum = gb_warp_sum(sum * whole_exp2(c - run.c));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = Stats{top, c, sum};
    __syncthreads();
    return join(WARPS, k, [&](int w) { return part[w]; });
}

// The sum alone of a block's share, by differences, for a maximum that is far.
template <typename T>
__device__ float far_sum(const Row<T>& row, float m, float k, bool with_edges, Stats* part) {
    float s = 0.0f;
    for (int i = row.lo + (int)threadIdx.x; i < row.hi; i += THREADS) {
        float2 v[Row<T>::P];
        Pack<T>::pairs(row.base[i], v);
        #pragma unroll
        for (int j = 0; j < Row<T>::P; ++j) s += fast_exp2((v[j].x - m) * k) + fast_exp2((v[j].y - m) * k);
    }
    if (with_edges && (int)threadIdx.x < row.edges()) s += fast_exp2((gb_up(row.x[row.edge(threadIdx.x)]) - m) * k);
    s = gb_warp_sum(s);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5].s = s;
    __syncthreads();
    float total = 0.0f;
    for (int w = 0; w < WARPS; ++w) total += part[w].s;
    return total;
}

// The gradient of this block's share of a row whose log-probability has the gradient `coef`;
// zeros from vocab to ld.  `out` lies across its vectors as the row does.
template <typename T>
__device__ void write_grad(const Row<T>& row, T* out, int ld, int target, float coef, Stats stats, const Base& base,
                           bool with_edges) {
    constexpr int N = Row<T>::N, P = Row<T>::P;
    // p = 2^(x k + c) / s; what k leaves out goes into s, as it is at the maximum
    const float k = base.k, c = stats.c, inv_temperature = (float)base.inv_temperature;
    const bool far = is_far(stats.m, k);
    const float left = far ? 0.0f : stats.m * base.rest;
    const float s = stats.s * (fabsf(left) < 0.001f ? 1.0f - left * 0.69314718f : fast_exp2(-left));
    const float scale = -coef * inv_temperature / s, hit = coef * inv_temperature;
    const float2 k2 = both(k), c2 = both(c), scale2 = both(scale);
    uint4* to = reinterpret_cast<uint4*>(out - row.skew);
    const int at = (target + row.skew) / N, place = (target + row.skew) % N;
    auto give = [&](int i, const uint4& q) {
        float2 v[P];
        Pack<T>::pairs(q, v);
        #pragma unroll
        for (int j = 0; j < P; ++j) {
            const float2 t = far ? make_float2((v[j].x - stats.m) * k, (v[j].y - stats.m) * k) : fma2(v[j], k2, c2);
            v[j] = mul2(exp2_2(t), scale2);
        }
        if (i == at) {
            #pragma unroll
            for (int j = 0; j < P; ++j) {
                if (2 * j == place) v[j].x += hit;
                if (2 * j + 1 == place) v[j].y += hit;
            }
        }
        __stcs(to + i, Pack<T>::back(v));            // not read here again: the rows keep the cache
    };
    int i = row.lo + (int)threadIdx.x;
    for (; i + (BATCH - 1) * THREADS < row.hi; i += BATCH * THREADS) {
        uint4 q[BATCH];
        #pragma unroll
        for (int u = 0; u < BATCH; ++u) q[u] = __ldcs(row.base + i + u * THREADS);
        #pragma unroll
        for (int u = 0; u < BATCH; ++u) give(i + u * THREADS, q[u]);
    }
    if (i < row.hi) {
        uint4 q[BATCH];
        #pragma unroll
        for (int u = 0; u < BATCH; ++u) if (i + u * THREADS < row.hi) q[u] = __ldcs(row.base + i + u * THREADS);
        #pragma unroll
        for (int u = 0; u < BATCH; ++u) if (i + u * THREADS < row.hi) give(i + u * THREADS, q[u]);
    }
    if (!with_edges) return;
    if ((int)threadIdx.x < row.edges()) {
        const int col = row.edge(threadIdx.x);
        const float x = gb_up(row.x[col]);
        const float g = fast_exp2(far ? (x - stats.m) * k : fmaf(x, k, c)) * scale;
        out[col] = gb_down<T>(col == target ? g + hit : g);
    }
    for (int col = row.vocab + threadIdx.x; col < ld; col += THREADS) out[col] = gb_down<T>(0.0f);
}

template <typename T>
__device__ void write_zeros(const Row<T>& row, T* out, int ld, bool with_edges) {
    uint4* to = reinterpret_cast<uint4*>(out - row.skew);
    for (int i = row.lo + (int)threadIdx.x; i < row.hi; i += THREADS) __stcs(to + i, make_uint4(0u, 0u, 0u, 0u));
    if (!with_edges) return;
    if ((int)threadIdx.x < row.edges()) out[row.edge(threadIdx.x)] = gb_down<T>(0.0f);
    for (int col = row.vocab + threadIdx.x; col < ld; col += THREADS) out[col] = gb_down<T>(0.0f);
}

// Sum over the block in 64 bits, in a fixed order, in every thread.
template <int COUNT>
__device__ double block_sum(double v) {
    __shared__ double part[COUNT / 32];
    v = gb_warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    double total = part[0];
    for (int w = 1; w < COUNT / 32; ++w) total += part[w];
    return total;
}

struct ForwardArgs {
    Rows rows;
    const long long* targets;
    Base base;
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
constexpr int SMALL = 1024;              // threads of the one-block kernels

// The reciprocal of the denominator, which every row's coefficient needs.
__global__ void __launch_bounds__(SMALL) policy_denominator_kernel(const ForwardArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the rows' first sweep needs nothing of this
    double d = 0.0;
    if (a.denominator) d = *a.denominator;
    else {
        for (long long r = threadIdx.x; r < a.rows.rows; r += SMALL) {
            const long long t = a.targets[r];
            if (t >= 0 && t < a.rows.vocab) d += a.weights ? (double)a.weights[r] : 1.0;
        }
        d = block_sum<SMALL>(d);
    }
    // where no token counts, loss and gradient are 0
    if (threadIdx.x == 0) *a.inv_denominator = d == 0.0 ? 0.0f : (float)(1.0 / d);
}

// One row a block, or a row a cluster where there are fewer rows than the SMs can hold blocks.
template <typename T, int MODE>
__global__ void __launch_bounds__(THREADS, 5) forward_kernel(const ForwardArgs a) {
    __shared__ Stats s_part[WARPS], s_block;
    __shared__ float s_coef;
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const long long r = blockIdx.x / parts;
    const bool first = rank == 0;
    const float k = a.base.k;
    const long long at = a.rows.offset(r);
    const T* x = static_cast<const T*>(a.rows.x) + at;
    const Row<T> row(x, a.rows.vocab, rank, parts);
    const long long target = a.targets[r];
    const float weight = (MODE == POLICY && a.weights) ? a.weights[r] : 1.0f;
    const bool counted = target >= 0 && target < a.rows.vocab && weight != 0.0f;
    T* out = a.grad ? static_cast<T*>(a.grad) + r * a.rows.ld : nullptr;
    if (!counted) {                      // so it is for the whole cluster
        if (first && threadIdx.x == 0) {
            a.logprobs[r] = 0.0f;
            if (a.stats) a.stats[r] = make_float2(0.0f, 1.0f);
            if (MODE == POLICY) {
                a.coef[r] = 0.0f;
                for (int q = 0; q < 3; ++q) a.terms[q * a.rows.rows + r] = 0.0f;
            }
        }
        if (out) write_zeros(row, out, a.rows.ld, first);
        // whoever waits for this launch may count on the one ahead of it
        if (MODE == POLICY && threadIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    Stats stats = row_stats(row, a.base, first, s_part);
    if (parts > 1) {
        if (threadIdx.x == 0) s_block = stats;
        cluster.sync();
        stats = join(parts, k, [&](int p) { return *cluster.map_shared_rank(&s_block, p); });
    }
    if (is_far(stats.m, k)) {            // the same in every block of the cluster
        stats.s = far_sum(row, stats.m, k, first, s_part);
        if (parts > 1) {
            cluster.sync();
            if (threadIdx.x == 0) s_block.s = stats.s;
            cluster.sync();
            stats.s = 0.0f;
            for (int p = 0; p < parts; ++p) stats.s += cluster.map_shared_rank(&s_block, p)->s;
        }
    }
    if (threadIdx.x == 0) {
        const float picked = gb_up(x[target]);
        float adv = 0.0f, old = 0.0f, ref = 0.0f;
        if (MODE == POLICY) {
            adv = a.advantages[r];
            old = a.old[r];
            if (a.ref) ref = a.ref[r];
        }
        // in 64 bits: the numbers are some 20 and their difference may be anything
        const double at_max = is_far(stats.m, k) ? (double)picked - (double)stats.m : (double)picked;
        const double exact = at_max * a.base.inv_temperature + (double)stats.c * 0.69314718055994530942 -
                             log((double)stats.s) - EXP2_LOW;
        const float logprob = exact > 0.0 ? 0.0f : (float)exact;
        if (first) {
            a.logprobs[r] = logprob;
            if (a.stats) a.stats[r] = make_float2(stats.m, stats.s);
        }
        if (MODE == POLICY) {
            const float ratio = expf(logprob - old);
            const float low = 1.0f - a.clip_low, high = 1.0f + a.clip_high;
            const bool outside = (adv > 0.0f && ratio > high) || (adv < 0.0f && ratio < low);
            const float raw = ratio * adv;
            float loss = -fminf(raw, fminf(fmaxf(ratio, low), high) * adv);
            if (raw != raw) loss = raw;                                  // a NaN stays one
            float d = outside ? 0.0f : -adv * ratio;
            float kl = 0.0f;
            if (a.ref) {
                const float gap = ref - logprob, e = expm1f(gap);
                kl = e - gap;
                loss += a.kl_coef * kl;
                d -= a.kl_coef * e;
            }
            asm volatile("griddepcontrol.wait;" ::: "memory");           // the denominator is there
            s_coef = weight * *reinterpret_cast<volatile float*>(a.inv_denominator) * d;
            if (first) {
                a.terms[r] = weight * loss;
                a.terms[a.rows.rows + r] = weight * kl;
                a.terms[2 * a.rows.rows + r] = outside ? weight : 0.0f;
                a.coef[r] = s_coef;
            }
        }
    }
    if (MODE == POLICY && out) {
        __syncthreads();
        const float coef = s_coef;
        if (coef == 0.0f) write_zeros(row, out, a.rows.ld, first);
        else write_grad(row, out, a.rows.ld, (int)target, coef, stats, a.base, first);
    }
    if (parts > 1) cluster.sync();       // no block leaves while another may read its result
}

// The three sums of terms times the reciprocal denominator.
struct FinishArgs {
    const float* terms;
    long long rows;
    const float* inv;
    float *loss, *kl, *clipped;
};
__global__ void __launch_bounds__(SMALL) policy_finish_kernel(const FinishArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    double acc[3] = {0.0, 0.0, 0.0};
    #pragma unroll 4
    for (long long r = threadIdx.x; r < a.rows; r += SMALL) {
        #pragma unroll
        for (int q = 0; q < 3; ++q) acc[q] += a.terms[q * a.rows + r];
    }
    const double inv = *a.inv;
    #pragma unroll
    for (int q = 0; q < 3; ++q) {
        acc[q] = block_sum<SMALL>(acc[q]);
        if (threadIdx.x == 0) *(q == 0 ? a.loss : q == 1 ? a.kl : a.clipped) = (float)(acc[q] * inv);
    }
}

struct GradArgs {
    Rows rows;
    const long long* targets;
    const float2* stats;
    const float* coef;                   // [rows]
    const float* upstream;               // one value that multiplies every coefficient, or null
    Base base;
    void* grad;
    int parts;                           // blocks a row
};

template <typename T>
__global__ void __launch_bounds__(THREADS) grad_kernel(const GradArgs a) {
    const float up = a.upstream ? *a.upstream : 1.0f;
    const long long r = blockIdx.x / a.parts;
    const int part = (int)(blockIdx.x - r * a.parts);
    const Row<T> row(static_cast<const T*>(a.rows.x) + a.rows.offset(r), a.rows.vocab, part, a.parts);
    T* out = static_cast<T*>(a.grad) + r * a.rows.ld;
    const long long target = a.targets[r];
    const float own = a.coef[r], coef = own * up;
    if (target < 0 || target >= a.rows.vocab || own == 0.0f || coef == 0.0f) write_zeros(row, out, a.rows.ld, part == 0);
    else {
        const float2 st = a.stats[r];
        write_grad(row, out, a.rows.ld, (int)target, coef, Stats{st.x, offset_for(st.x, a.base.k), st.y}, a.base, part == 0);
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
__global__ void __launch_bounds__(SMALL) preference_kernel(const PreferenceArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = SMALL / 32;
    auto begin = [&](int s) {
        long long v = a.offsets ? a.offsets[s] : s * a.length;
        return v < 0 ? 0LL : (v > a.rows ? a.rows : v);      // whatever the offsets hold, rows are in range
    };
    for (int s = warp; s < a.sequences; s += warps) {
        const long long lo = begin(s), hi = begin(s + 1);
        double sum = 0.0, tokens = 0.0;
        #pragma unroll 8
        for (long long r = lo + lane; r < hi; r += 32) sum += a.logprobs[r];
        if (a.average) {
            #pragma unroll 8
            for (long long r = lo + lane; r < hi; r += 32)
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
    for (int p = threadIdx.x; p < pairs; p += SMALL) {
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
    loss = block_sum<SMALL>(loss);                          // its barriers also publish seq_coef
    if (threadIdx.x == 0) *a.loss = (float)(loss / pairs);
    for (long long r = threadIdx.x; r < begin(0); r += SMALL) a.coef[r] = 0.0f;
    for (long long r = begin(a.sequences) + threadIdx.x; r < a.rows; r += SMALL) a.coef[r] = 0.0f;
    for (int s = warp; s < a.sequences; s += warps) {
        const float c = a.seq_coef[s];
        for (long long r = begin(s) + lane; r < begin(s + 1); r += 32) a.coef[r] = c;
    }
}

// Blocks that share a row: as many as keep the SMs busy (five blocks fit on each), but not less
// than two vectors for every thread of them, and no more than a cluster may have.
int parts_for(long long rows, int vocab, int width) {
    const long long vectors = (long long)vocab * width / 16;
    int parts = 1;
    while (parts < 8 && rows * parts * 2 <= 148 * 5 && vectors >= (long long)parts * 2 * THREADS * 2) parts *= 2;
    return parts;
}

// A launch of clusters of `parts` blocks.  `early`: it may begin before the launch ahead of it is done,
// which it waits for where it needs it.
template <typename K, typename A>
int start(K kernel, long long grid, int threads, int parts, bool early, cudaStream_t stream, A args) {
    if (grid > 0x7fffffff) return (int)cudaErrorInvalidValue;
    cudaLaunchAttribute attr[2] = {};
    int n = 0;
    if (parts > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = (unsigned)parts;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (early) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)grid);
    config.blockDim = dim3(threads);
    config.stream = stream;
    config.attrs = attr;
    config.numAttrs = n;
    return (int)cudaLaunchKernelEx(&config, kernel, args);
}

template <int MODE>
int start_forward(int dtype, const ForwardArgs& a, bool early, cudaStream_t stream) {
    const int parts = parts_for(a.rows.rows, a.rows.vocab, dtype == GB_F32 ? 4 : 2);
    const long long grid = a.rows.rows * parts;
    if (dtype == GB_F32) return start(forward_kernel<float, MODE>, grid, THREADS, parts, early, stream, a);
    if (dtype == GB_BF16) return start(forward_kernel<__nv_bfloat16, MODE>, grid, THREADS, parts, early, stream, a);
    if (dtype == GB_F16) return start(forward_kernel<__half, MODE>, grid, THREADS, parts, early, stream, a);
    return (int)cudaErrorInvalidValue;
}

Base base_of(double temperature) {
    const double k = 1.4426950408889634074 / temperature;
    return Base{(float)k, (float)(k - (double)(float)k), 1.0 / temperature};
}

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
                                 double temperature, float* logprobs, float* stats, cudaStream_t stream) {
    ForwardArgs a = {};
    a.rows = Rows{logits, batch_stride, row_stride, inner, rows, vocab, ld};
    if (bad(a.rows)) return (int)cudaErrorInvalidValue;
    a.targets = targets; a.base = base_of(temperature); a.logprobs = logprobs;
    a.stats = reinterpret_cast<float2*>(stats);
    return start_forward<LOGPROBS>(dtype, a, false, stream);
}

// scratch: 3 * rows + 1 floats.  loss, kl, clipped (share): one float each.  ref, weights and denominator may be
// null; grad null: backward is gb_logprob_grad with `coef` and `stats` (null where grad is given).
extern "C" int gb_policy_loss(int dtype, const void* logits, long long batch_stride, long long row_stride,
                              long long inner, long long rows, int vocab, int ld, const long long* targets,
                              double temperature, const float* old, const float* advantages, const float* ref,
                              const float* weights, const float* denominator, float clip_low, float clip_high,
                              float kl_coef, float* logprobs, float* stats, float* coef, float* scratch,
                              float* loss, float* kl, float* clipped, void* grad, cudaStream_t stream) {
    ForwardArgs a = {};
    a.rows = Rows{logits, batch_stride, row_stride, inner, rows, vocab, ld};
    if (bad(a.rows)) return (int)cudaErrorInvalidValue;
    a.targets = targets; a.base = base_of(temperature); a.logprobs = logprobs;
    a.stats = reinterpret_cast<float2*>(stats);
    a.old = old; a.advantages = advantages; a.ref = ref; a.weights = weights; a.denominator = denominator;
    a.clip_low = clip_low; a.clip_high = clip_high; a.kl_coef = kl_coef;
    a.coef = coef; a.terms = scratch; a.inv_denominator = scratch + 3 * rows; a.grad = grad;
    int err = start(policy_denominator_kernel, 1, SMALL, 1, false, stream, a);
    if (err) return err;
    if ((err = start_forward<POLICY>(dtype, a, true, stream))) return err;
    const FinishArgs f = {scratch, rows, scratch + 3 * rows, loss, kl, clipped};
    return start(policy_finish_kernel, 1, SMALL, 1, true, stream, f);
}

extern "C" int gb_logprob_grad(int dtype, const void* logits, long long batch_stride, long long row_stride,
                               long long inner, long long rows, int vocab, int ld, const long long* targets,
                               double temperature, const float* stats, const float* coef, const float* upstream,
                               void* grad, cudaStream_t stream) {
    GradArgs a = {};
    a.rows = Rows{logits, batch_stride, row_stride, inner, rows, vocab, ld};
    if (bad(a.rows)) return (int)cudaErrorInvalidValue;
    a.targets = targets; a.stats = reinterpret_cast<const float2*>(stats); a.coef = coef; a.upstream = upstream;
    a.base = base_of(temperature); a.grad = grad;
    a.parts = parts_for(rows, vocab, dtype == GB_F32 ? 4 : 2);
    const long long grid = rows * a.parts;
    if (dtype == GB_F32) return start(grad_kernel<float>, grid, THREADS, 1, false, stream, a);
    if (dtype == GB_BF16) return start(grad_kernel<__nv_bfloat16>, grid, THREADS, 1, false, stream, a);
    if (dtype == GB_F16) return start(grad_kernel<__half>, grid, THREADS, 1, false, stream, a);
    return (int)cudaErrorInvalidValue;
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
    return start(preference_kernel, 1, SMALL, 1, true, stream, a);
}
