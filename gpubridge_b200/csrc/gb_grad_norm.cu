// The global norm of many gradient tensors, the scaling that clips them, and an AdamW step that
// takes the scaling along.
//
//   norm = sqrt(sum of g^2)  (or max |g|),   coef = min(1, max_norm / (norm + 1e-6))
//
// The list of tensors travels in the kernel's parameters (20 KB of the 32 KB a launch may carry),
// so a call copies nothing to the device and can be captured in a CUDA graph.  Tensors are cut
// into chunks of CHUNK values; block b takes chunks b, b + grid, ..., finds a chunk's tensor by
// bisection and leaves one partial result; a second launch of one block adds the partials in
// index order, so the result does not depend on scheduling.  Squares and sums are in 64 bits:
// no gradient that is finite in its own type makes the norm overflow or vanish, and the 64-bit
// units of a B200 keep up with the memory.  Bound by the one read of the gradients: 134 M fp32
// values in 111 tensors take 84 us (6.4 TB/s; 92 us with one vector a thread under way instead of
// four).  The clipped AdamW step of 124 M values takes 635 us with its norm; reading the gradients
// twice and everything else once is 617 us at the rate of a copy.  Walking the update from the
// gradients that the norm read last, to find them in L2, gained nothing: the other streams push
// them out.
#include "gb_vec.cuh"

namespace {

constexpr int MAX_TENSORS = 1024;
constexpr int THREADS = 256;
constexpr long long CHUNK = 32768;

struct TensorList {
    void* ptr[MAX_TENSORS];
    long long n[MAX_TENSORS];
    int first[MAX_TENSORS];            // index of the tensor's first chunk
    int count;
    int chunks;
};

// The tensor that holds chunk c.  Tensors without values own no chunk and are not in the list.
__device__ __forceinline__ int owner_of(const TensorList& list, int c) {
    int lo = 0, hi = list.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (list.first[mid] <= c) lo = mid; else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double larger(double a, double b) {     // NaN wins
    return (a > b || a != a) ? a : b;
}

template <bool MAX>
__device__ __forceinline__ void take(double& acc, float v) {
    if (MAX) acc = larger(fabs((double)v), acc);
    else { const double d = v; acc = fma(d, d, acc); }
}

template <typename T, bool MAX>
__global__ void __launch_bounds__(THREADS)
norm_kernel(const __grid_constant__ TensorList list, double* __restrict__ part) {
    double acc = 0.0;
    for (int c = blockIdx.x; c < list.chunks; c += gridDim.x) {
        const int t = owner_of(list, c);
        const long long lo = (long long)(c - list.first[t]) * CHUNK;
        const long long left = list.n[t] - lo;
        const int n = (int)(left < CHUNK ? left : CHUNK);
        const T* p = static_cast<const T*>(list.ptr[t]) + lo;
        constexpr int BYTES = 8 * (int)sizeof(T);
        int head = (int)((BYTES - (int)(reinterpret_cast<uintptr_t>(p) & (BYTES - 1))) & (BYTES - 1)) / (int)sizeof(T);
        if (head > n) head = n;
        const int vecs = (n - head) / 8;
        int i = threadIdx.x;
        for (; i + 3 * THREADS < vecs; i += 4 * THREADS) {           // four vectors under way
            Raw8<T> raw[4];
            #pragma unroll
            for (int u = 0; u < 4; ++u) raw[u].load(p + head + (i + u * THREADS) * 8);
            #pragma unroll
            for (int u = 0; u < 4; ++u) {
                float v[8];
                raw[u].get(v);
                #pragma unroll
                for (int j = 0; j < 8; ++j) take<MAX>(acc, v[j]);
            }
        }
        for (; i < vecs; i += THREADS) {
            Raw8<T> raw;
            float v[8];
            raw.load(p + head + i * 8);
            raw.get(v);
            #pragma unroll
            for (int j = 0; j < 8; ++j) take<MAX>(acc, v[j]);
        }
        for (int i = threadIdx.x; i < head; i += THREADS) take<MAX>(acc, gb_up(p[i]));
        for (int i = head + vecs * 8 + threadIdx.x; i < n; i += THREADS) take<MAX>(acc, gb_up(p[i]));
    }
    __shared__ double warp_part[THREADS / 32];
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const double other = __shfl_xor_sync(0xffffffffu, acc, o);
        acc = MAX ? larger(acc, other) : acc + other;
    }
    if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        double total = warp_part[0];
        for (int w = 1; w < THREADS / 32; ++w) total = MAX ? larger(total, warp_part[w]) : total + warp_part[w];
        part[blockIdx.x] = total;
    }
}

// result[0] = norm of the gradients times `scale`, result[1] = the factor that clips them.
template <bool MAX>
__global__ void __launch_bounds__(THREADS)
finish_kernel(const double* __restrict__ part, int parts, double scale, double max_norm,
              float* __restrict__ result) {
    double acc = 0.0;
    for (int i = threadIdx.x; i < parts; i += THREADS) acc = MAX ? larger(part[i], acc) : acc + part[i];
    __shared__ double warp_part[THREADS / 32];
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const double other = __shfl_xor_sync(0xffffffffu, acc, o);
        acc = MAX ? larger(acc, other) : acc + other;
    }
    if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        double total = warp_part[0];
        for (int w = 1; w < THREADS / 32; ++w) total = MAX ? larger(total, warp_part[w]) : total + warp_part[w];
        const double norm = (MAX ? total : sqrt(total)) * fabs(scale);
        const double coef = max_norm / (norm + 1e-6);
        result[0] = (float)norm;
        result[1] = coef > 1.0 ? 1.0f : (float)coef;           // a NaN stays one
    }
}

// result[1] from a norm that was found elsewhere (result[0], device memory).
__global__ void coef_kernel(const float* __restrict__ norm, double max_norm, float* __restrict__ result) {
    const double n = norm[0], coef = max_norm / (n + 1e-6);
    result[0] = norm[0];
    result[1] = coef > 1.0 ? 1.0f : (float)coef;
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
scale_kernel(const __grid_constant__ TensorList list, const float* __restrict__ coef_at) {
    const float coef = *coef_at;
    if (coef == 1.0f) return;                                   // within the limit: nothing to write
    for (int c = blockIdx.x; c < list.chunks; c += gridDim.x) {
        const int t = owner_of(list, c);
        const long long lo = (long long)(c - list.first[t]) * CHUNK;
        const long long left = list.n[t] - lo;
        const int n = (int)(left < CHUNK ? left : CHUNK);
        T* p = static_cast<T*>(list.ptr[t]) + lo;
        constexpr int BYTES = 8 * (int)sizeof(T);
        int head = (int)((BYTES - (int)(reinterpret_cast<uintptr_t>(p) & (BYTES - 1))) & (BYTES - 1)) / (int)sizeof(T);
        if (head > n) head = n;
        const int vecs = (n - head) / 8;
        for (int i = threadIdx.x; i < vecs; i += THREADS) {
            Raw8<T> raw;
            float v[8];
            raw.load(p + head + i * 8);
            raw.get(v);
            #pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= coef;
            gb_store8(p + head + i * 8, v);
        }
        for (int i = threadIdx.x; i < head; i += THREADS) p[i] = gb_down<T>(gb_up(p[i]) * coef);
        for (int i = head + vecs * 8 + threadIdx.x; i < n; i += THREADS) p[i] = gb_down<T>(gb_up(p[i]) * coef);
    }
}

// False where the list cannot be taken: too many tensors, or more chunks than an int counts.
bool make_list(void* const* ptrs, const long long* sizes, int count, TensorList& list) {
    if (count < 0 || count > MAX_TENSORS) return false;
    long long chunks = 0;
    list.count = 0;
    for (int i = 0; i < count; ++i) {
        if (sizes[i] < 0) return false;
        if (sizes[i] == 0) continue;
        if (!ptrs[i]) return false;
        list.ptr[list.count] = ptrs[i];
        list.n[list.count] = sizes[i];
        list.first[list.count] = (int)chunks;
        ++list.count;
        chunks += (sizes[i] + CHUNK - 1) / CHUNK;
        if (chunks > 0x7fffffff) return false;
    }
    list.chunks = (int)chunks;
    return true;
}

constexpr int MAX_BLOCKS = 148 * 8;

int grid_for(int chunks) { return chunks < MAX_BLOCKS ? (chunks > 0 ? chunks : 1) : MAX_BLOCKS; }

struct AdamState {                     // that of gb_adamw_span
    unsigned int arrived;
    unsigned int pad;
    float step;
    float pad2;
};

struct AdamScalars {                   // 1 - beta and log(beta) come from the host's 64 bits
    float beta1, beta2, one_minus_beta1, one_minus_beta2, eps, lr, decay;
    double log_beta1, log_beta2;
};

// The arithmetic of torch.optim.AdamW on gradients times `grad_scale` times *coef_at.
__global__ void __launch_bounds__(256)
adamw_clipped_kernel(float* __restrict__ p, float* __restrict__ g, float* __restrict__ m,
                     float* __restrict__ v, size_t n, AdamState* state, const AdamScalars s,
                     float grad_scale, const float* __restrict__ coef_at, int zero_grad) {
    __shared__ float s_step_size, s_rsqrt_bc2;
    if (threadIdx.x == 0) {
        const float step = *reinterpret_cast<volatile float*>(&state->step) + 1.0f;
        __threadfence();
        // the last block to have read the old step count publishes the new one
        if (atomicAdd(&state->arrived, 1u) + 1u == gridDim.x) {
            state->arrived = 0u;
            *reinterpret_cast<volatile float*>(&state->step) = step;
        }
        const double bc1 = -expm1((double)step * s.log_beta1), bc2 = -expm1((double)step * s.log_beta2);
        s_step_size = (float)((double)s.lr / bc1);
        s_rsqrt_bc2 = (float)(1.0 / sqrt(bc2));
    }
    __syncthreads();
    const float step_size = s_step_size, rsqrt_bc2 = s_rsqrt_bc2;
    const float scale = grad_scale * *coef_at;
    auto update = [&](float& pe, float ge, float& me, float& ve) {
        const float grad = ge * scale;
        me = s.beta1 * me + s.one_minus_beta1 * grad;
        ve = s.beta2 * ve + s.one_minus_beta2 * grad * grad;
        pe = pe * s.decay - step_size * (me / (sqrtf(ve) * rsqrt_bc2 + s.eps));
    };
    const size_t nvec = n >> 2;
    const size_t tid = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    const size_t nth = (size_t)gridDim.x * blockDim.x;
    float4* p4 = reinterpret_cast<float4*>(p);
    float4* g4 = reinterpret_cast<float4*>(g);
    float4* m4 = reinterpret_cast<float4*>(m);
    float4* v4 = reinterpret_cast<float4*>(v);
    for (size_t i = tid; i < nvec; i += nth) {
        float4 pp = p4[i], gg = g4[i], mm = m4[i], vv = v4[i];
        update(pp.x, gg.x, mm.x, vv.x);
        update(pp.y, gg.y, mm.y, vv.y);
        update(pp.z, gg.z, mm.z, vv.z);
        update(pp.w, gg.w, mm.w, vv.w);
        p4[i] = pp; m4[i] = mm; v4[i] = vv;
        if (zero_grad) g4[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (size_t i = (nvec << 2) + tid; i < n; i += nth) {
        float pe = p[i], me = m[i], ve = v[i];
        update(pe, g[i], me, ve);
        p[i] = pe; m[i] = me; v[i] = ve;
        if (zero_grad) g[i] = 0.f;
    }
}

}  // namespace

// How many partial results (doubles) a call over `count` tensors leaves.
extern "C" int gb_grad_norm_parts(void* const* ptrs, const long long* sizes, int count) {
    TensorList list;
    if (!make_list(ptrs, sizes, count, list)) return -1;
    return grid_for(list.chunks);
}

extern "C" int gb_grad_norm_max_tensors() { return MAX_TENSORS; }

// Partial sums of squares (or largest magnitudes) of up to 1024 tensors of one type into
// part[0 .. gb_grad_norm_parts).  Tensors may start at any multiple of their values' size.
extern "C" int gb_grad_norm_partial(int dtype, int maximum, void* const* ptrs, const long long* sizes,
                                    int count, double* part, cudaStream_t stream) {
    TensorList list;
    if (!make_list(ptrs, sizes, count, list)) return (int)cudaErrorInvalidValue;
    const int grid = grid_for(list.chunks);
#define GB_NORM(T) (maximum ? norm_kernel<T, true><<<grid, THREADS, 0, stream>>>(list, part) \
                            : norm_kernel<T, false><<<grid, THREADS, 0, stream>>>(list, part))
    if (dtype == GB_F32) GB_NORM(float);
    else if (dtype == GB_BF16) GB_NORM(__nv_bfloat16);
    else if (dtype == GB_F16) GB_NORM(__half);
    else return (int)cudaErrorInvalidValue;
#undef GB_NORM
    return (int)cudaGetLastError();
}

// result[0] = norm * |scale|, result[1] = min(1, max_norm / (result[0] + 1e-6)).
extern "C" int gb_grad_norm_finish(int maximum, const double* part, int parts, double scale,
                                   double max_norm, float* result, cudaStream_t stream) {
    if (maximum) finish_kernel<true><<<1, THREADS, 0, stream>>>(part, parts, scale, max_norm, result);
    else finish_kernel<false><<<1, THREADS, 0, stream>>>(part, parts, scale, max_norm, result);
    return (int)cudaGetLastError();
}

extern "C" int gb_grad_clip_coef(const float* norm, double max_norm, float* result, cudaStream_t stream) {
    coef_kernel<<<1, 1, 0, stream>>>(norm, max_norm, result);
    return (int)cudaGetLastError();
}

// Every value of the tensors times *coef; nothing is touched where *coef is 1.
extern "C" int gb_grad_scale(int dtype, void* const* ptrs, const long long* sizes, int count,
                             const float* coef, cudaStream_t stream) {
    TensorList list;
    if (!make_list(ptrs, sizes, count, list)) return (int)cudaErrorInvalidValue;
    const int grid = grid_for(list.chunks);
    if (dtype == GB_F32) scale_kernel<float><<<grid, THREADS, 0, stream>>>(list, coef);
    else if (dtype == GB_BF16) scale_kernel<__nv_bfloat16><<<grid, THREADS, 0, stream>>>(list, coef);
    else if (dtype == GB_F16) scale_kernel<__half><<<grid, THREADS, 0, stream>>>(list, coef);
    else return (int)cudaErrorInvalidValue;
    return (int)cudaGetLastError();
}

// gb_adamw_span over whole buffers, with every gradient times grad_scale times *coef.
extern "C" int gb_adamw_clipped(float* p, float* g, float* m, float* v, size_t n, void* state,
                                double lr, double beta1, double beta2, double eps, double weight_decay,
                                float grad_scale, const float* coef, int zero_grad, cudaStream_t stream) {
    AdamScalars s;
    s.beta1 = (float)beta1; s.beta2 = (float)beta2;
    s.one_minus_beta1 = (float)(1.0 - beta1); s.one_minus_beta2 = (float)(1.0 - beta2);
    s.eps = (float)eps; s.lr = (float)lr; s.decay = (float)(1.0 - lr * weight_decay);
    s.log_beta1 = log(beta1); s.log_beta2 = log(beta2);
    size_t blocks = (n / 4 + 256 * 4 - 1) / (256 * 4);
    if (blocks < 1) blocks = 1;
    if (blocks > 148 * 8) blocks = 148 * 8;
    adamw_clipped_kernel<<<(int)blocks, 256, 0, stream>>>(p, g, m, v, n, static_cast<AdamState*>(state),
                                                          s, grad_scale, coef, zero_grad);
    return (int)cudaGetLastError();
}
