// The join of a block with the residual stream, with the norms on either side of it, in one pass:
//
//   v      = norm(update; post_weight, post_bias)        (or update itself)
//   stream = residual + scale * gate * v                 rounded once, in the stream's type
//   normed = norm(stream; weight, bias)                  (or nothing: the block that follows has its own)
//
// with norm(x) = x / sqrt(mean(x^2) + eps) * w  (rms)  or  (x - mean) / sqrt(var + eps) * w + b.
// The gate has one value a channel, for all rows or for each group of consecutive rows (a
// sequence).  Backward, with dr the gradient that reaches the stream:
//
//   dr = d_stream + norm'(d_normed),   d_residual = dr,   d_gate = sum over rows of scale * dr * v
//   dv = scale * gate * dr,            d_update = norm'(dv)
//   norm'(g; x^, r) = r * (g w - mean(g w x^) x^ [- mean(g w)])
//
// Bound by memory: forward reads residual and update and writes stream and normed, backward reads
// both gradients, the stream and the update and writes two gradients.  A block owns a row, its
// values stay in registers between the reductions, and it walks several rows so that the
// gradients of the parameters, sums over all rows, are gathered in registers; each block leaves
// its partial sums and a second launch adds them in index order.
#include "gb_vec.cuh"

namespace {

struct JoinArgs {
    const void* residual;              // rows of d values, row_stride apart
    const void* update;
    long long residual_stride, update_stride;
    void* stream;                      // [rows, d]
    void* normed;                      // [rows, d] or null
    float4* stats;                     // [rows]: mean and 1 / deviation of the update, of the stream
    const void *weight, *bias, *post_weight, *post_bias, *gate;     // null where absent
    const void *d_stream, *d_normed;   // [rows, d] or null
    void *d_residual, *d_update;
    float* part;                       // [workers][sums][d]
    float* gate_part;                  // [workers + groups - 1][d]
    long long rows, group_rows;        // rows of one gate group
    int d, layer, param_code, gate_code, next;
    float scale, eps;
};

constexpr int MAX_THREADS = 512;
constexpr int MAX_WARPS = MAX_THREADS / 32;

// Sums over the block's threads; the buffers alternate, so one barrier a reduction is enough.
struct Reducer {
    float2* buffer;                    // [2][MAX_WARPS]
    int parity = 0;
    __device__ float2 sum(float2 v) {
        v.x = gb_warp_sum(v.x);
        v.y = gb_warp_sum(v.y);
        const int warps = blockDim.x >> 5;
        if (warps == 1) return v;
        float2* b = buffer + parity * MAX_WARPS;
        parity ^= 1;
        if ((threadIdx.x & 31) == 0) b[threadIdx.x >> 5] = v;
        __syncthreads();
        float2 total = b[0];
        for (int w = 1; w < warps; ++w) { total.x += b[w].x; total.y += b[w].y; }
        return total;
    }
};

// A thread's place in a row: vector k of NV starts at column (k * blockDim.x + threadIdx.x) * VEC.
template <int VEC, int NV>
struct Lane {
    int col[NV];
    bool ok[NV];
    __device__ explicit Lane(int d) {
        #pragma unroll
        for (int k = 0; k < NV; ++k) {
            col[k] = (k * (int)blockDim.x + (int)threadIdx.x) * VEC;
            ok[k] = col[k] < d;                     // d is a multiple of VEC
        }
    }
    template <typename T>
    __device__ void load(const T* row, float (&v)[NV][VEC]) const {
        if constexpr (VEC == 8) {
            Raw8<T> raw[NV];
            #pragma unroll
            for (int k = 0; k < NV; ++k) if (ok[k]) raw[k].load(row + col[k]);
            #pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (ok[k]) raw[k].get(v[k]);
                else {
                    #pragma unroll
                    for (int j = 0; j < VEC; ++j) v[k][j] = 0.0f;
                }
            }
        } else {
            #pragma unroll
            for (int k = 0; k < NV; ++k) v[k][0] = ok[k] ? gb_up(row[col[k]]) : 0.0f;
        }
    }
    template <typename T>
    __device__ void store(T* row, const float (&v)[NV][VEC]) const {
        #pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (!ok[k]) continue;
            if constexpr (VEC == 8) gb_store8(row + col[k], v[k]);
            else row[col[k]] = gb_down<T>(v[k][0]);
        }
    }
    // a parameter's values in this thread's columns; `otherwise` where there is no such parameter
    __device__ void param(const void* p, int code, float otherwise, float (&v)[NV][VEC]) const {
        #pragma unroll
        for (int k = 0; k < NV; ++k) {
            #pragma unroll
            for (int j = 0; j < VEC; ++j) v[k][j] = (p && ok[k]) ? gb_read(p, code, col[k] + j) : otherwise;
        }
    }
    __device__ void sums(float* row, const float (&v)[NV][VEC]) const {
        #pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (!ok[k]) continue;
            #pragma unroll
            for (int j = 0; j < VEC; ++j) row[col[k] + j] = v[k][j];
        }
    }
};

__device__ __forceinline__ size_t param_bytes(int code) { return code == GB_F32 ? 4 : 2; }

// Mean (0 for rms) and 1 / deviation of a row.
template <int VEC, int NV>
__device__ float2 row_stats(const Lane<VEC, NV>& lane, const float (&v)[NV][VEC], int d, int layer,
                            float eps, Reducer& reduce) {
    const float inv = 1.0f / (float)d;
    float mean = 0.0f;
    if (layer) {
        float s = 0.0f;
        #pragma unroll
        for (int k = 0; k < NV; ++k) {
            #pragma unroll
            for (int j = 0; j < VEC; ++j) s += v[k][j];
        }
        mean = reduce.sum(make_float2(s, 0.0f)).x * inv;
    }
    float q = 0.0f;
    #pragma unroll
    for (int k = 0; k < NV; ++k) {
        #pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float c = lane.ok[k] ? v[k][j] - mean : 0.0f;
            q += c * c;
        }
    }
    const float var = reduce.sum(make_float2(q, 0.0f)).x * inv;
    return make_float2(mean, 1.0f / sqrtf(var + eps));
}

template <typename TS, typename TU, typename TY, int VEC, int NV>
__global__ void __launch_bounds__(MAX_THREADS) join_fwd_kernel(const JoinArgs a) {
    __shared__ float2 buffer[2 * MAX_WARPS];
    Reducer reduce{buffer};
    const Lane<VEC, NV> lane(a.d);
    float w[NV][VEC], b[NV][VEC], pw[NV][VEC], pb[NV][VEC], gate[NV][VEC];
    lane.param(a.weight, a.param_code, 1.0f, w);
    lane.param(a.bias, a.param_code, 0.0f, b);
    lane.param(a.post_weight, a.param_code, 1.0f, pw);
    lane.param(a.post_bias, a.param_code, 0.0f, pb);
    lane.param(nullptr, 0, 1.0f, gate);
    long long group = -1;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float u[NV][VEC], r[NV][VEC];
        lane.load(static_cast<const TU*>(a.update) + row * a.update_stride, u);
        lane.load(static_cast<const TS*>(a.residual) + row * a.residual_stride, r);
        if (a.gate) {
            const long long mine = row / a.group_rows;
            if (mine != group) {
                group = mine;
                lane.param(static_cast<const char*>(a.gate) + group * a.d * param_bytes(a.gate_code),
                           a.gate_code, 1.0f, gate);
            }
        }
        float4 st = make_float4(0.0f, 1.0f, 0.0f, 1.0f);
        if (a.post_weight) {
            const float2 s = row_stats(lane, u, a.d, a.layer, a.eps, reduce);
            st.x = s.x; st.y = s.y;
            #pragma unroll
            for (int k = 0; k < NV; ++k) {
                #pragma unroll
                for (int j = 0; j < VEC; ++j) u[k][j] = (u[k][j] - s.x) * s.y * pw[k][j] + pb[k][j];
            }
        }
        #pragma unroll
        for (int k = 0; k < NV; ++k) {
            #pragma unroll
            for (int j = 0; j < VEC; ++j) {
                // the norm that follows is that of the stream as it is stored
                r[k][j] = gb_up(gb_down<TS>(fmaf(a.scale * gate[k][j], u[k][j], r[k][j])));
                if (!lane.ok[k]) r[k][j] = 0.0f;
            }
        }
        lane.store(static_cast<TS*>(a.stream) + row * a.d, r);
        if (a.next) {
            const float2 s = row_stats(lane, r, a.d, a.layer, a.eps, reduce);
            st.z = s.x; st.w = s.y;
            #pragma unroll
            for (int k = 0; k < NV; ++k) {
                #pragma unroll
                for (int j = 0; j < VEC; ++j) r[k][j] = (r[k][j] - s.x) * s.y * w[k][j] + b[k][j];
            }
            lane.store(static_cast<TY*>(a.normed) + row * a.d, r);
        }
        if (a.stats && threadIdx.x == 0) a.stats[row] = st;
    }
}

// Worker c owns the rows [first_row(c), first_row(c + 1)); owner_of is its inverse.
__host__ __device__ __forceinline__ long long first_row(long long c, long long rows, long long workers) {
    return c * rows / workers;
}
__host__ __device__ __forceinline__ long long owner_of(long long row, long long rows, long long workers) {
    return ((row + 1) * workers - 1) / rows;
}

// r * (g - mean(g x^) x^ [- mean(g)]) over a row, g given in place.
template <int VEC, int NV>
__device__ void norm_backward(const Lane<VEC, NV>& lane, float (&g)[NV][VEC], const float (&hat)[NV][VEC],
                              float rstd, int d, int layer, Reducer& reduce) {
    float2 s = make_float2(0.0f, 0.0f);
    #pragma unroll
    for (int k = 0; k < NV; ++k) {
        #pragma unroll
        for (int j = 0; j < VEC; ++j) {
            s.x += g[k][j] * hat[k][j];
            s.y += g[k][j];
        }
    }
    s = reduce.sum(s);
    const float inv = 1.0f / (float)d, m1 = s.x * inv, m0 = layer ? s.y * inv : 0.0f;
    #pragma unroll
    for (int k = 0; k < NV; ++k) {
        #pragma unroll
        for (int j = 0; j < VEC; ++j)
            g[k][j] = lane.ok[k] ? rstd * (g[k][j] - m0 - hat[k][j] * m1) : 0.0f;
    }
}

// One block is one worker.  part[worker] holds, one behind the other, the sums of d_weight,
// d_bias, d_post_weight, d_post_bias that exist.  Worker c and gate group g meet in slot c + g of
// gate_part: along the rows one of the two grows by one at a time, so no two pairs share a slot.
template <typename TS, typename TU, typename TY, int VEC, int NV>
__global__ void __launch_bounds__(MAX_THREADS) join_bwd_kernel(const JoinArgs a) {
    __shared__ float2 buffer[2 * MAX_WARPS];
    Reducer reduce{buffer};
    const Lane<VEC, NV> lane(a.d);
    float w[NV][VEC], pw[NV][VEC], pb[NV][VEC], gate[NV][VEC];
    float dw[NV][VEC], db[NV][VEC], dpw[NV][VEC], dpb[NV][VEC], dg[NV][VEC];
    lane.param(a.weight, a.param_code, 1.0f, w);
    lane.param(a.post_weight, a.param_code, 1.0f, pw);
    lane.param(a.post_bias, a.param_code, 0.0f, pb);
    lane.param(nullptr, 0, 1.0f, gate);
    lane.param(nullptr, 0, 0.0f, dw);
    lane.param(nullptr, 0, 0.0f, db);
    lane.param(nullptr, 0, 0.0f, dpw);
    lane.param(nullptr, 0, 0.0f, dpb);
    lane.param(nullptr, 0, 0.0f, dg);
    const bool needs_update = a.post_weight || a.gate;
    const long long worker = blockIdx.x;
    const long long lo = first_row(worker, a.rows, gridDim.x), hi = first_row(worker + 1, a.rows, gridDim.x);
    long long group = -1;
    for (long long row = lo; row < hi; ++row) {
        if (a.gate) {
            const long long mine = row / a.group_rows;
            if (mine != group) {
                if (group >= 0) lane.sums(a.gate_part + (worker + group) * a.d, dg);
                group = mine;
                lane.param(nullptr, 0, 0.0f, dg);
                lane.param(static_cast<const char*>(a.gate) + group * a.d * param_bytes(a.gate_code),
                           a.gate_code, 1.0f, gate);
            }
        }
        float dr[NV][VEC], u[NV][VEC];
        const float4 st = a.stats[row];
        if (a.d_stream) lane.load(static_cast<const TS*>(a.d_stream) + row * a.d, dr);
        else lane.param(nullptr, 0, 0.0f, dr);
        if (needs_update) lane.load(static_cast<const TU*>(a.update) + row * a.update_stride, u);
        if (a.d_normed) {
            float g[NV][VEC], hat[NV][VEC];
            lane.load(static_cast<const TY*>(a.d_normed) + row * a.d, g);
            lane.load(static_cast<const TS*>(a.stream) + row * a.d, hat);
            #pragma unroll
            for (int k = 0; k < NV; ++k) {
                #pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    hat[k][j] = (hat[k][j] - st.z) * st.w;
                    dw[k][j] += g[k][j] * hat[k][j];
                    db[k][j] += g[k][j];
                    g[k][j] *= w[k][j];
                }
            }
            norm_backward(lane, g, hat, st.w, a.d, a.layer, reduce);
            #pragma unroll
            for (int k = 0; k < NV; ++k) {
                #pragma unroll
                for (int j = 0; j < VEC; ++j) dr[k][j] += g[k][j];
            }
        }
        if (a.d_residual) lane.store(static_cast<TS*>(a.d_residual) + row * a.d, dr);
        #pragma unroll
        for (int k = 0; k < NV; ++k) {
            #pragma unroll
            for (int j = 0; j < VEC; ++j) dr[k][j] *= a.scale;
        }
        if (needs_update) {
            #pragma unroll
            for (int k = 0; k < NV; ++k) {
                #pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    u[k][j] = (u[k][j] - st.x) * st.y;            // the update itself without a post norm
                    dg[k][j] += dr[k][j] * (u[k][j] * pw[k][j] + pb[k][j]);
                    dr[k][j] *= gate[k][j];
                    dpw[k][j] += dr[k][j] * u[k][j];
                    dpb[k][j] += dr[k][j];
                    dr[k][j] *= pw[k][j];
                }
            }
            if (a.post_weight) norm_backward(lane, dr, u, st.y, a.d, a.layer, reduce);
        }
        lane.store(static_cast<TU*>(a.d_update) + row * a.d, dr);
    }
    if (a.gate && group >= 0) lane.sums(a.gate_part + (worker + group) * a.d, dg);
    const int sums = (a.d_normed ? (a.bias ? 2 : 1) : 0) + (a.post_weight ? (a.post_bias ? 2 : 1) : 0);
    float* mine = a.part + worker * sums * a.d;
    if (a.d_normed) { lane.sums(mine, dw); mine += a.d; }
    if (a.d_normed && a.bias) { lane.sums(mine, db); mine += a.d; }
    if (a.post_weight) { lane.sums(mine, dpw); mine += a.d; }
    if (a.post_weight && a.post_bias) lane.sums(mine, dpb);
}

struct SumArgs {
    const float* part;
    const float* gate_part;
    void* out[4];                      // one for each sum, in the order of part
    void* gate_out;                    // [groups][d]
    long long rows, group_rows, groups, workers;
    int d, sums, param_code, gate_code;
};

// Column sums of the partial results: 32 columns a block, SLICES threads share a column.
constexpr int SLICES = 16;
__global__ void __launch_bounds__(32 * SLICES) join_sum_kernel(const SumArgs a) {
    const int col = blockIdx.y * 32 + threadIdx.x;
    const long long which = blockIdx.x;
    const float* base;
    long long lo = 0, hi = a.workers;
    size_t stride;
    if (which < a.sums) {
        base = a.part + which * a.d;
        stride = (size_t)a.sums * a.d;
    } else {
        const long long g = which - a.sums;
        lo = owner_of(g * a.group_rows, a.rows, a.workers);
        hi = owner_of((g + 1) * a.group_rows - 1, a.rows, a.workers) + 1;
        base = a.gate_part + g * a.d;
        stride = a.d;
    }
    float acc = 0.0f;
    if (col < a.d) for (long long c = lo + threadIdx.y; c < hi; c += SLICES) acc += base[c * stride + col];
    __shared__ float slice[SLICES][33];
    slice[threadIdx.y][threadIdx.x] = acc;
    __syncthreads();
    if (threadIdx.y == 0 && col < a.d) {
        float total = slice[0][threadIdx.x];
        for (int s = 1; s < SLICES; ++s) total += slice[s][threadIdx.x];
        if (which < a.sums) gb_write(a.out[which], a.param_code, col, total);
        else gb_write(a.gate_out, a.gate_code, (size_t)(which - a.sums) * a.d + col, total);
    }
}

constexpr int MAX_WIDTH = 8192;

// Threads of a block for rows of d values in vectors of vec.
int threads_for(int d, int vec) {
    int t = (d + vec - 1) / vec;
    t = (t + 31) / 32 * 32;
    return t < MAX_THREADS ? t : MAX_THREADS;
}

int workers_for(long long rows, int threads) {
    // enough blocks to fill the SMs at the registers these kernels take, and no more: each leaves
    // a row of partial sums
    int per_sm = 512 / threads;
    if (per_sm < 1) per_sm = 1;
    if (per_sm > 8) per_sm = 8;
    const long long most = 148LL * per_sm;
    return (int)(rows < most ? rows : most);
}

template <typename TS, typename TU, typename TY>
int launch(bool forward, int vec, const JoinArgs& a, cudaStream_t s) {
    const int t = threads_for(a.d, vec);
    const int nv = (a.d + t * vec - 1) / (t * vec);
    long long grid;
    if (forward) {
        long long cap = 148LL * (2048 / t < 16 ? 2048 / t : 16);
        grid = a.rows < cap ? a.rows : cap;
    } else grid = workers_for(a.rows, t);
#define GB_JOIN(VEC, NV) (forward ? join_fwd_kernel<TS, TU, TY, VEC, NV><<<(int)grid, t, 0, s>>>(a) \
                                  : join_bwd_kernel<TS, TU, TY, VEC, NV><<<(int)grid, t, 0, s>>>(a))
    if (vec == 8) {
        if (nv <= 1) GB_JOIN(8, 1);
        else if (nv <= 2) GB_JOIN(8, 2);
        else return (int)cudaErrorInvalidValue;
    } else {
        if (nv <= 1) GB_JOIN(1, 1);
        else if (nv <= 4) GB_JOIN(1, 4);
        else if (nv <= 16) GB_JOIN(1, 16);
        else return (int)cudaErrorInvalidValue;
    }
#undef GB_JOIN
    return (int)cudaGetLastError();
}

int dispatch(bool forward, int s, int u, int y, int vec, const JoinArgs& a, cudaStream_t stream) {
    if (a.rows <= 0 || a.d <= 0 || a.d > MAX_WIDTH || (vec != 1 && vec != 8) || a.d % vec) return (int)cudaErrorInvalidValue;
#define GB_TYPES(A, B, C, TA, TB, TC) if (s == A && u == B && y == C) return launch<TA, TB, TC>(forward, vec, a, stream);
    GB_TYPES(GB_F32, GB_F32, GB_F32, float, float, float)
    GB_TYPES(GB_F32, GB_BF16, GB_BF16, float, __nv_bfloat16, __nv_bfloat16)
    GB_TYPES(GB_F32, GB_F16, GB_F16, float, __half, __half)
    GB_TYPES(GB_BF16, GB_BF16, GB_BF16, __nv_bfloat16, __nv_bfloat16, __nv_bfloat16)
    GB_TYPES(GB_F16, GB_F16, GB_F16, __half, __half, __half)
#undef GB_TYPES
    return (int)cudaErrorInvalidValue;
}

}  // namespace

// Types: codes of gb_vec.cuh; (stream, update, normed) is one of (f32, f32, f32), (f32, low, low),
// (low, low, low) with low bf16 or fp16.  vec = 8 wants every row to begin on a vector boundary
// (32 bytes of f32, 16 of the others) and d to be a multiple of 8; vec = 1 takes any.  d <= 8192.
extern "C" int gb_residual_norm_fwd(int s, int u, int y, int vec, const void* residual,
                                    long long residual_stride, const void* update, long long update_stride,
                                    void* stream, void* normed, float* stats, const void* weight,
                                    const void* bias, const void* post_weight, const void* post_bias,
                                    int param_code, const void* gate, int gate_code, long long rows,
                                    long long group_rows, int d, int layer, float scale, float eps,
                                    cudaStream_t cuda_stream) {
    JoinArgs a = {};
    a.residual = residual; a.update = update; a.residual_stride = residual_stride; a.update_stride = update_stride;
    a.stream = stream; a.normed = normed; a.stats = reinterpret_cast<float4*>(stats);
    a.weight = weight; a.bias = bias; a.post_weight = post_weight; a.post_bias = post_bias; a.gate = gate;
    a.param_code = param_code; a.gate_code = gate_code; a.rows = rows; a.group_rows = group_rows;
    a.d = d; a.layer = layer; a.next = normed != nullptr; a.scale = scale; a.eps = eps;
    return dispatch(true, s, u, y, vec, a, cuda_stream);
}

// Workers (blocks) of a backward call: part holds workers * sums * d floats, gate_part
// (workers + groups - 1) * d.
extern "C" int gb_residual_norm_workers(long long rows, int d, int vec) {
    return workers_for(rows, threads_for(d, vec));
}

// The stream, both gradients (either may be null) and the outputs are [rows, d] without gaps;
// d_residual may be null.  out: the gradients of weight, bias, post_weight, post_bias that exist
// (the first two only where d_normed is given), in this order; gate_out [rows / group_rows, d].
extern "C" int gb_residual_norm_bwd(int s, int u, int y, int vec, const void* d_stream, const void* d_normed,
                                    const void* stream, const void* update, long long update_stride,
                                    const float* stats, const void* weight, const void* bias,
                                    const void* post_weight, const void* post_bias, int param_code,
                                    const void* gate, int gate_code, void* d_residual, void* d_update,
                                    float* part, float* gate_part, void* out0, void* out1, void* out2,
                                    void* out3, void* gate_out, long long rows, long long group_rows,
                                    int d, int layer, float scale, cudaStream_t cuda_stream) {
    JoinArgs a = {};
    a.update = update; a.update_stride = update_stride; a.stream = const_cast<void*>(stream);
    a.stats = reinterpret_cast<float4*>(const_cast<float*>(stats));
    a.weight = weight; a.bias = bias; a.post_weight = post_weight; a.post_bias = post_bias; a.gate = gate;
    a.d_stream = d_stream; a.d_normed = d_normed; a.d_residual = d_residual; a.d_update = d_update;
    a.part = part; a.gate_part = gate_part; a.param_code = param_code; a.gate_code = gate_code;
    a.rows = rows; a.group_rows = group_rows; a.d = d; a.layer = layer; a.scale = scale;
    const int err = dispatch(false, s, u, y, vec, a, cuda_stream);
    if (err) return err;
    SumArgs q = {};
    q.part = part; q.gate_part = gate_part; q.gate_out = gate_out;
    q.out[0] = out0; q.out[1] = out1; q.out[2] = out2; q.out[3] = out3;
    q.rows = rows; q.group_rows = group_rows; q.groups = gate ? rows / group_rows : 0;
    q.workers = gb_residual_norm_workers(rows, d, vec);
    q.d = d; q.param_code = param_code; q.gate_code = gate_code;
    q.sums = (d_normed ? (bias ? 2 : 1) : 0) + (post_weight ? (post_bias ? 2 : 1) : 0);
    const long long what = q.sums + q.groups;
    if (what == 0) return 0;
    if (what > 0x7fffffff) return (int)cudaErrorInvalidValue;
    join_sum_kernel<<<dim3((unsigned)what, (d + 31) / 32), dim3(32, SLICES), 0, cuda_stream>>>(q);
    return (int)cudaGetLastError();
}
