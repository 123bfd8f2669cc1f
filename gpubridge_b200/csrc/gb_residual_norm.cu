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
// both gradients, the stream and the update and writes two gradients.  A block owns a row, eight
// columns a thread; their values stay in registers between the reductions while the next rows are
// already on their way to shared memory.  A block walks several rows, so that the gradients of the
// parameters, sums over all rows, are gathered in registers; it leaves its partial sums and a
// second launch adds them in index order.
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
    int d, layer, param_code, gate_code, next, stages;
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
    __device__ float sum(float v) {
        v = gb_warp_sum(v);
        const int warps = blockDim.x >> 5;
        if (warps == 1) return v;
        float* b = reinterpret_cast<float*>(buffer + parity * MAX_WARPS);
        parity ^= 1;
        if ((threadIdx.x & 31) == 0) b[threadIdx.x >> 5] = v;
        __syncthreads();
        float total = b[0];
        for (int w = 1; w < warps; ++w) total += b[w];
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
    __device__ void store(T* row, const float (&v)[NV][VEC]) const {
        #pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (!ok[k]) continue;
            if constexpr (VEC == 8) gb_store8(row + col[k], v[k]);
            else row[col[k]] = gb_down<T>(v[k][0]);
        }
    }
    __device__ static void fill(float value, float (&v)[NV][VEC]) {
        #pragma unroll
        for (int k = 0; k < NV; ++k) {
            #pragma unroll
            for (int j = 0; j < VEC; ++j) v[k][j] = value;
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
            if constexpr (VEC == 8) gb_store8(row + col[k], v[k]);
            else row[col[k]] = v[k][0];
        }
    }
};

// Rows of one tensor on their way to this thread's registers.  Each thread copies the values that
// it will use itself, STAGES - 1 rows ahead, into its own places in shared memory (cp.async), so
// the loads of several rows are in flight while a row is reduced, no register holds them and no
// barrier guards them.  Single values of two bytes cannot be copied so: they are read when used.
template <typename T, int VEC, int NV>
struct Feed {
    static constexpr bool STAGED = VEC == 8 || sizeof(T) == 4;
    static constexpr int PIECE = VEC == 8 ? 16 : 4;                     // bytes of one copy
    static constexpr int PIECES = VEC == 8 ? (int)sizeof(T) / 2 : 1;    // copies a vector
    static constexpr int BYTES = STAGED ? NV * PIECES * PIECE : 0;      // a thread and stage
    const T* base;
    long long stride;
    uint32_t at;                       // shared address of this thread's first piece of stage 0
    uint32_t stage_bytes;
    __device__ void place(const void* p, long long row_stride, uint32_t region, uint32_t per_stage) {
        base = static_cast<const T*>(p);
        stride = row_stride;
        at = region + threadIdx.x * PIECE;
        stage_bytes = per_stage;
    }
    __device__ void fetch(const Lane<VEC, NV>& lane, long long row, int stage) const {
        if constexpr (STAGED) {
            const T* from = base + row * stride;
            #pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (!lane.ok[k]) continue;
                #pragma unroll
                for (int h = 0; h < PIECES; ++h) {
                    const uint32_t to = at + stage * stage_bytes + (k * PIECES + h) * blockDim.x * PIECE;
                    const T* src = from + lane.col[k] + h * (16 / (int)sizeof(T));
                    if constexpr (PIECE == 16)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(to), "l"(src) : "memory");
                    else
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" :: "r"(to), "l"(src) : "memory");
                }
            }
        }
    }
    __device__ void get(const Lane<VEC, NV>& lane, long long row, int stage, float (&v)[NV][VEC]) const {
        #pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (!lane.ok[k]) {
                #pragma unroll
                for (int j = 0; j < VEC; ++j) v[k][j] = 0.0f;
                continue;
            }
            if constexpr (VEC == 8) {
                #pragma unroll
                for (int h = 0; h < PIECES; ++h) {
                    const uint32_t from = at + stage * stage_bytes + (k * PIECES + h) * blockDim.x * PIECE;
                    uint4 q;
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "r"(from) : "memory");
                    if constexpr (sizeof(T) == 4) {
                        v[k][4 * h] = __uint_as_float(q.x); v[k][4 * h + 1] = __uint_as_float(q.y);
                        v[k][4 * h + 2] = __uint_as_float(q.z); v[k][4 * h + 3] = __uint_as_float(q.w);
                    } else {
                        Raw8<T> raw;
                        raw.q = q;
                        raw.get(v[k]);
                    }
                }
            } else if constexpr (STAGED) {
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[k][0])
                             : "r"(at + stage * stage_bytes + k * blockDim.x * PIECE) : "memory");
            } else {
                v[k][0] = gb_up(base[row * stride + lane.col[k]]);
            }
        }
    }
};

__device__ __forceinline__ void feed_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// waits until at most `ahead` of the groups this thread committed are under way
__device__ __forceinline__ void feed_wait(int ahead) {
    switch (ahead) {
        case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
        case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
        case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
        default: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
    }
}
constexpr int MAX_STAGES = 4;

__device__ __forceinline__ size_t param_bytes(int code) { return code == GB_F32 ? 4 : 2; }

// Mean (0 for rms) and 1 / deviation of a row.  The variance is that of the centred values, which
// are at hand: a second reduction instead of a difference of large numbers.
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
        mean = reduce.sum(s) * inv;
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
    const float var = reduce.sum(q) * inv;
    return make_float2(mean, 1.0f / sqrtf(var + eps));
}

// The gate's values for a row; they are read again where a row begins another group.
template <int VEC, int NV>
struct Gate {
    float v[NV][VEC];
    long long group = -1, left = 0;    // rows until the next group
    __device__ Gate() { Lane<VEC, NV>::fill(1.0f, v); }
    // true where the row begins a group other than the last one's
    __device__ bool move(const JoinArgs& a, const Lane<VEC, NV>& lane, long long row, long long step) {
        left -= step;
        if (left > 0 && group >= 0) return false;
        const long long mine = row / a.group_rows;
        left = (mine + 1) * a.group_rows - row;
        if (mine == group) return false;
        group = mine;
        lane.param(static_cast<const char*>(a.gate) + group * a.d * param_bytes(a.gate_code), a.gate_code, 1.0f, v);
        return true;
    }
};

extern __shared__ __align__(16) char join_shared[];

template <typename TS, typename TU, typename TY, int VEC, int NV>
__global__ void __launch_bounds__(MAX_THREADS) join_fwd_kernel(const JoinArgs a) {
    __shared__ float2 buffer[2 * MAX_WARPS];
    Reducer reduce{buffer};
    const Lane<VEC, NV> lane(a.d);
    Feed<TS, VEC, NV> from_residual;
    Feed<TU, VEC, NV> from_update;
    constexpr int BYTES = Feed<TS, VEC, NV>::BYTES + Feed<TU, VEC, NV>::BYTES;
    const uint32_t shared = (uint32_t)__cvta_generic_to_shared(join_shared), per_stage = BYTES * blockDim.x;
    from_residual.place(a.residual, a.residual_stride, shared, per_stage);
    from_update.place(a.update, a.update_stride, shared + Feed<TS, VEC, NV>::BYTES * blockDim.x, per_stage);
    const long long step = gridDim.x;
    auto fetch = [&](long long row, int stage) {
        if (row < a.rows) {
            from_residual.fetch(lane, row, stage);
            from_update.fetch(lane, row, stage);
        }
        feed_commit();
    };
    for (int i = 0; i < a.stages - 1; ++i) fetch(blockIdx.x + i * step, i);
    float w[NV][VEC], b[NV][VEC], pw[NV][VEC], pb[NV][VEC];
    lane.param(a.weight, a.param_code, 1.0f, w);
    lane.param(a.bias, a.param_code, 0.0f, b);
    lane.param(a.post_weight, a.param_code, 1.0f, pw);
    lane.param(a.post_bias, a.param_code, 0.0f, pb);
    Gate<VEC, NV> gate;
    int stage = 0;
    for (long long row = blockIdx.x; row < a.rows; row += step) {
        const int ahead = stage == 0 ? a.stages - 1 : stage - 1;
        fetch(row + (a.stages - 1) * step, ahead);
        feed_wait(a.stages - 1);
        float u[NV][VEC], r[NV][VEC];
        from_update.get(lane, row, stage, u);
        from_residual.get(lane, row, stage, r);
        stage = stage + 1 == a.stages ? 0 : stage + 1;
        if (a.gate) gate.move(a, lane, row, step);
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
                r[k][j] = gb_up(gb_down<TS>(fmaf(a.scale * gate.v[k][j], u[k][j], r[k][j])));
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
    if (layer) s = reduce.sum(s);
    else s.x = reduce.sum(s.x);
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
// NEXT: the following norm's gradient takes part; OWN: the update has a norm or a gate of its own.
template <typename TS, typename TU, typename TY, int VEC, int NV, bool NEXT, bool OWN>
__global__ void __launch_bounds__(MAX_THREADS) join_bwd_kernel(const JoinArgs a) {
    __shared__ float2 buffer[2 * MAX_WARPS];
    Reducer reduce{buffer};
    const Lane<VEC, NV> lane(a.d);
    using FS = Feed<TS, VEC, NV>;
    using FU = Feed<TU, VEC, NV>;
    using FY = Feed<TY, VEC, NV>;
    FS from_grad, from_stream;
    FU from_update;
    FY from_normed;
    constexpr int BYTES = FS::BYTES + (NEXT ? FS::BYTES + FY::BYTES : 0) + (OWN ? FU::BYTES : 0);
    const uint32_t per_stage = BYTES * blockDim.x;
    uint32_t region = (uint32_t)__cvta_generic_to_shared(join_shared);
    from_grad.place(a.d_stream, a.d, region, per_stage);
    region += FS::BYTES * blockDim.x;
    if (NEXT) {
        from_stream.place(a.stream, a.d, region, per_stage);
        region += FS::BYTES * blockDim.x;
        from_normed.place(a.d_normed, a.d, region, per_stage);
        region += FY::BYTES * blockDim.x;
    }
    if (OWN) from_update.place(a.update, a.update_stride, region, per_stage);
    const long long worker = blockIdx.x;
    const long long lo = first_row(worker, a.rows, gridDim.x), hi = first_row(worker + 1, a.rows, gridDim.x);
    auto fetch = [&](long long row, int stage) {
        if (row < hi) {
            if (a.d_stream) from_grad.fetch(lane, row, stage);
            if (NEXT) {
                from_stream.fetch(lane, row, stage);
                from_normed.fetch(lane, row, stage);
            }
            if (OWN) from_update.fetch(lane, row, stage);
        }
        feed_commit();
    };
    for (int i = 0; i < a.stages - 1; ++i) fetch(lo + i, i);
    float w[NV][VEC], pw[NV][VEC], pb[NV][VEC];
    float dw[NV][VEC], db[NV][VEC], dpw[NV][VEC], dpb[NV][VEC], dg[NV][VEC];
    lane.param(a.weight, a.param_code, 1.0f, w);
    lane.param(a.post_weight, a.param_code, 1.0f, pw);
    lane.param(a.post_bias, a.param_code, 0.0f, pb);
    Gate<VEC, NV> gate;
    lane.fill(0.0f, dw);
    lane.fill(0.0f, db);
    lane.fill(0.0f, dpw);
    lane.fill(0.0f, dpb);
    lane.fill(0.0f, dg);
    int stage = 0;
    for (long long row = lo; row < hi; ++row) {
        const int ahead = stage == 0 ? a.stages - 1 : stage - 1;
        fetch(row + a.stages - 1, ahead);
        const float4 st = a.stats[row];
        if (OWN && a.gate) {
            const long long before = gate.group;
            if (gate.move(a, lane, row, 1) && before >= 0) {
                lane.sums(a.gate_part + (worker + before) * a.d, dg);
                lane.fill(0.0f, dg);
            }
        }
        feed_wait(a.stages - 1);
        float dr[NV][VEC];
        if (a.d_stream) from_grad.get(lane, row, stage, dr);
        else lane.fill(0.0f, dr);
        if (NEXT) {
            float g[NV][VEC], hat[NV][VEC];
            from_normed.get(lane, row, stage, g);
            from_stream.get(lane, row, stage, hat);
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
        if (OWN) {
            float u[NV][VEC];
            from_update.get(lane, row, stage, u);
            #pragma unroll
            for (int k = 0; k < NV; ++k) {
                #pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    u[k][j] = (u[k][j] - st.x) * st.y;            // the update itself without a post norm
                    dg[k][j] += dr[k][j] * (u[k][j] * pw[k][j] + pb[k][j]);
                    dr[k][j] *= gate.v[k][j];
                    dpw[k][j] += dr[k][j] * u[k][j];
                    dpb[k][j] += dr[k][j];
                    dr[k][j] *= pw[k][j];
                }
            }
            if (a.post_weight) norm_backward(lane, dr, u, st.y, a.d, a.layer, reduce);
        }
        lane.store(static_cast<TU*>(a.d_update) + row * a.d, dr);
        stage = stage + 1 == a.stages ? 0 : stage + 1;
    }
    if (OWN && a.gate && gate.group >= 0) lane.sums(a.gate_part + (worker + gate.group) * a.d, dg);
    const int sums = (NEXT ? (a.bias ? 2 : 1) : 0) + (a.post_weight ? (a.post_bias ? 2 : 1) : 0);
    float* mine = a.part + worker * sums * a.d;
    if (NEXT) { lane.sums(mine, dw); mine += a.d; }
    if (NEXT && a.bias) { lane.sums(mine, db); mine += a.d; }
    if (OWN && a.post_weight) { lane.sums(mine, dpw); mine += a.d; }
    if (OWN && a.post_weight && a.post_bias) lane.sums(mine, dpb);
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

// Threads of a block for rows of d values in vectors of vec, and its rounds of vectors: a single
// round of eight columns a thread up to 4096 columns, two from there on; single values in up to
// four rounds of 256 threads, then sixteen of 512.
struct Shape { int threads, rounds; };
Shape shape_of(int d, int vec) {
    const int vectors = (d + vec - 1) / vec, most = vec == 8 || vectors > 1024 ? MAX_THREADS : 256;
    int t = (vectors + 31) / 32 * 32;
    if (t > most) t = most;
    return Shape{t, (vectors + t - 1) / t};
}

// Blocks an SM holds at the 128 registers that 512 threads may have; each leaves a row of partial
// sums, so there are no more than fill the SMs.
int blocks_per_sm(int threads) {
    const int n = 512 / threads;
    return n < 1 ? 1 : n > 8 ? 8 : n;
}

int workers_for(long long rows, int threads) {
    const long long most = 148LL * blocks_per_sm(threads);
    return (int)(rows < most ? rows : most);
}

// Stages that fit beside one another in an SM's 227 KB.
int stages_for(int bytes_per_stage, int blocks) {
    int n = bytes_per_stage ? (int)((220 << 10) / blocks / bytes_per_stage) : MAX_STAGES;
    return n < 1 ? 1 : n > MAX_STAGES ? MAX_STAGES : n;
}

template <typename K>
int start(K kernel, int grid, int threads, int bytes_per_stage, int blocks, JoinArgs a, cudaStream_t s) {
    a.stages = stages_for(bytes_per_stage, blocks);
    const int shared = a.stages * bytes_per_stage;
    if (shared > (40 << 10)) {                       // more than a launch may take unasked, with the static part
        const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared);
        if (err != cudaSuccess) return (int)err;
    }
    kernel<<<grid, threads, shared, s>>>(a);
    return (int)cudaGetLastError();
}

template <typename TS, typename TU, typename TY, int VEC, int NV>
int launch_shaped(bool forward, int threads, const JoinArgs& a, cudaStream_t s) {
    constexpr int S = Feed<TS, VEC, NV>::BYTES, U = Feed<TU, VEC, NV>::BYTES, Y = Feed<TY, VEC, NV>::BYTES;
    const int blocks = blocks_per_sm(threads);
    const int grid = workers_for(a.rows, threads);
    if (forward) return start(join_fwd_kernel<TS, TU, TY, VEC, NV>, grid, threads, (S + U) * threads, blocks, a, s);
    const bool next = a.d_normed, own = a.post_weight || a.gate;
    if (next && own) return start(join_bwd_kernel<TS, TU, TY, VEC, NV, true, true>, grid, threads, (2 * S + Y + U) * threads, blocks, a, s);
    if (next) return start(join_bwd_kernel<TS, TU, TY, VEC, NV, true, false>, grid, threads, (2 * S + Y) * threads, blocks, a, s);
    return start(join_bwd_kernel<TS, TU, TY, VEC, NV, false, true>, grid, threads, (S + U) * threads, blocks, a, s);
}

template <typename TS, typename TU, typename TY>
int launch(bool forward, int vec, const JoinArgs& a, cudaStream_t s) {
    const Shape shape = shape_of(a.d, vec);
    if (vec == 8) {
        if (shape.rounds == 1) return launch_shaped<TS, TU, TY, 8, 1>(forward, shape.threads, a, s);
        return launch_shaped<TS, TU, TY, 8, 2>(forward, shape.threads, a, s);
    }
    if (shape.rounds <= 1) return launch_shaped<TS, TU, TY, 1, 1>(forward, shape.threads, a, s);
    if (shape.rounds <= 4) return launch_shaped<TS, TU, TY, 1, 4>(forward, shape.threads, a, s);
    return launch_shaped<TS, TU, TY, 1, 16>(forward, shape.threads, a, s);
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
    return workers_for(rows, shape_of(d, vec).threads);
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
