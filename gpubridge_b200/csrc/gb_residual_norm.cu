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
    int d, layer, param_code, gate_code, next, slots;
    float scale, eps;
};

constexpr int MAX_THREADS = 512;
constexpr int MAX_WARPS = MAX_THREADS / 32;

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

// Sums of Q values over the block's threads, one barrier a reduction: the buffers alternate.
// Within a warp the values are exchanged for one another before they are added, so that Q = 1, 2,
// 4 cost five, five and six shuffles.
struct Reducer {
    float* buffer;                     // [2][MAX_WARPS][4]
    int warps, parity;
    __device__ explicit Reducer(float* b) : buffer(b), warps((int)blockDim.x >> 5), parity(0) {
        for (int i = threadIdx.x; i < 2 * MAX_WARPS * 4; i += blockDim.x) b[i] = 0.0f;
        __syncthreads();
    }
    template <int Q>
    __device__ void sum(float (&v)[Q]) {
        static_assert(Q == 1 || Q == 2 || Q == 4, "values of one reduction");
        const int lane = threadIdx.x & 31;
        float mine;
        if constexpr (Q == 4) {
            const bool upper = lane & 16;
            float a = upper ? v[2] : v[0], b = upper ? v[3] : v[1];
            const float sa = upper ? v[0] : v[2], sb = upper ? v[1] : v[3];
            a += __shfl_xor_sync(0xffffffffu, sa, 16);
            b += __shfl_xor_sync(0xffffffffu, sb, 16);
            const bool second = lane & 8;
            mine = second ? b : a;
            mine += __shfl_xor_sync(0xffffffffu, second ? a : b, 8);
        } else if constexpr (Q == 2) {
            const bool upper = lane & 16;
            mine = upper ? v[1] : v[0];
            mine += __shfl_xor_sync(0xffffffffu, upper ? v[0] : v[1], 16);
        } else mine = v[0];
        #pragma unroll
        for (int step = Q == 4 ? 4 : Q == 2 ? 8 : 16; step > 0; step >>= 1)
            mine += __shfl_xor_sync(0xffffffffu, mine, step);
        float* b = buffer + parity * MAX_WARPS * 4;
        parity ^= 1;
        if (lane % (32 / Q) == 0) b[(threadIdx.x >> 5) * Q + lane / (32 / Q)] = mine;
        if (warps == 1) __syncwarp(); else __syncthreads();
        // all partial results, four warps at a time (there are zeros behind the last)
        const float4* b4 = reinterpret_cast<const float4*>(b);
        #pragma unroll
        for (int q = 0; q < Q; ++q) v[q] = 0.0f;
        for (int w = 0; w < warps; w += 4) {
            #pragma unroll
            for (int i = 0; i < Q; ++i) {
                const float4 f = b4[(w / 4) * Q + i];
                const float e[4] = {f.x, f.y, f.z, f.w};
                #pragma unroll
                for (int j = 0; j < 4; ++j) v[(4 * i + j) % Q] += e[j];
            }
        }
    }
};

// A thread's place in a row: vector k of NV starts at column (k * blockDim.x + threadIdx.x) * VEC.
// Its values are held in pairs: value e of the thread is that of vector e / VEC.
template <int VEC, int NV>
struct Lane {
    static constexpr int E = VEC * NV, P = (E + 1) / 2;
    int col[NV];
    bool ok[NV];
    __device__ explicit Lane(int d) {
        #pragma unroll
        for (int k = 0; k < NV; ++k) {
            col[k] = (k * (int)blockDim.x + (int)threadIdx.x) * VEC;
            ok[k] = col[k] < d;                     // d is a multiple of VEC
        }
    }
    __device__ static float& at(float2 (&v)[P], int e) { return e & 1 ? v[e / 2].y : v[e / 2].x; }
    __device__ static float at(const float2 (&v)[P], int e) { return e & 1 ? v[e / 2].y : v[e / 2].x; }
    template <typename T>
    __device__ void store(T* row, const float2 (&v)[P]) const {
        #pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (!ok[k]) continue;
            if constexpr (VEC == 8) {
                float f[8];
                #pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = at(v, k * 8 + j);
                gb_store8(row + col[k], f);
            } else row[col[k]] = gb_down<T>(at(v, k));
        }
    }
    __device__ static void fill(float value, float2 (&v)[P]) {
        #pragma unroll
        for (int i = 0; i < P; ++i) v[i] = both(value);
    }
    // 0 in the places of no column
    __device__ void mask(float2 (&v)[P]) const {
        #pragma unroll
        for (int e = 0; e < E; ++e) if (!ok[e / VEC]) at(v, e) = 0.0f;
        if (E & 1) v[P - 1].y = 0.0f;
    }
    // a parameter's values in this thread's columns; `otherwise` where there is no such parameter
    __device__ void param(const void* p, int code, float otherwise, float2 (&v)[P]) const {
        fill(otherwise, v);
        if (!p) return;
        #pragma unroll
        for (int e = 0; e < E; ++e) if (ok[e / VEC]) at(v, e) = gb_read(p, code, col[e / VEC] + e % VEC);
    }
};

// Rows of one tensor on their way to this thread's registers.  Each thread copies the values that
// it will use itself into its own places in shared memory (cp.async), as many rows ahead as there
// are slots, so the loads of several rows are in flight while a row is reduced, no register holds
// them and no barrier guards them.  Single values of two bytes cannot be copied so: they are read
// when used.
template <typename T, int VEC, int NV>
struct Feed {
    static constexpr bool STAGED = VEC == 8 || sizeof(T) == 4;
    static constexpr int PIECE = VEC == 8 ? 16 : 4;                     // bytes of one copy
    static constexpr int PIECES = VEC == 8 ? (int)sizeof(T) / 2 : 1;    // copies a vector
    static constexpr int BYTES = STAGED ? NV * PIECES * PIECE : 0;      // a thread and slot
    using L = Lane<VEC, NV>;
    const T* base;
    long long stride;
    uint32_t at;                       // shared address of this thread's first piece of slot 0
    __device__ void place(const void* p, long long row_stride, uint32_t region) {
        base = static_cast<const T*>(p);
        stride = row_stride;
        at = region + threadIdx.x * PIECE;
    }
    __device__ void fetch(const L& lane, long long row, uint32_t slot_offset) const {
        if constexpr (STAGED) {
            const T* from = base + row * stride;
            #pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (!lane.ok[k]) continue;
                #pragma unroll
                for (int h = 0; h < PIECES; ++h) {
                    const uint32_t to = at + slot_offset + (k * PIECES + h) * blockDim.x * PIECE;
                    const T* src = from + lane.col[k] + h * (16 / (int)sizeof(T));
                    if constexpr (PIECE == 16)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(to), "l"(src) : "memory");
                    else
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" :: "r"(to), "l"(src) : "memory");
                }
            }
        }
    }
    __device__ void get(const L& lane, long long row, uint32_t slot_offset, float2 (&v)[L::P]) const {
        if (L::E & 1) v[L::P - 1].y = 0.0f;
        #pragma unroll
        for (int k = 0; k < NV; ++k) {
            if constexpr (VEC == 8) {
                float f[8] = {};
                if (lane.ok[k]) {
                    #pragma unroll
                    for (int h = 0; h < PIECES; ++h) {
                        const uint32_t from = at + slot_offset + (k * PIECES + h) * blockDim.x * PIECE;
                        uint4 q;
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "r"(from) : "memory");
                        if constexpr (sizeof(T) == 4) {
                            f[4 * h] = __uint_as_float(q.x); f[4 * h + 1] = __uint_as_float(q.y);
                            f[4 * h + 2] = __uint_as_float(q.z); f[4 * h + 3] = __uint_as_float(q.w);
                        } else {
                            Raw8<T> raw;
                            raw.q = q;
                            raw.get(f);
                        }
                    }
                }
                #pragma unroll
                for (int j = 0; j < 8; ++j) L::at(v, k * 8 + j) = f[j];
            } else {
                float f = 0.0f;
                if (lane.ok[k]) {
                    if constexpr (STAGED)
                        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f)
                                     : "r"(at + slot_offset + k * blockDim.x * PIECE) : "memory");
                    else f = gb_up(base[row * stride + lane.col[k]]);
                }
                L::at(v, k) = f;
            }
        }
    }
};

__device__ __forceinline__ void feed_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// waits until at most `behind` of the groups this thread committed are under way
__device__ __forceinline__ void feed_wait(int behind) {
    switch (behind) {
        case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
        case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
        case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
        case 3: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
        case 4: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
        case 5: asm volatile("cp.async.wait_group 5;" ::: "memory"); break;
        default: asm volatile("cp.async.wait_group 6;" ::: "memory"); break;
    }
}
constexpr int MAX_SLOTS = 8;

// Worker c owns the rows [first_row(c), first_row(c + 1)); owner_of is its inverse.
__host__ __device__ __forceinline__ long long first_row(long long c, long long rows, long long workers) {
    return c * rows / workers;
}
__host__ __device__ __forceinline__ long long owner_of(long long row, long long rows, long long workers) {
    return ((row + 1) * workers - 1) / rows;
}

// A worker's walk over its rows: up to R at a time, all of one gate group, with the rows behind
// them under way.  One group of copies a row, in the rows' order, so a wait for all but the last
// slots - R groups is a wait for the rows at hand.
template <int R>
struct Walk {
    long long row, hi, fetched, group, group_end, group_rows;
    int slots, slot, count, fetch_slot;
    bool gated;
    __device__ Walk(const JoinArgs& a)
        : row(first_row(blockIdx.x, a.rows, gridDim.x)), hi(first_row(blockIdx.x + 1LL, a.rows, gridDim.x)),
          fetched(row), group(-1), group_end(hi), group_rows(a.group_rows), slots(a.slots), slot(0), count(0),
          fetch_slot(0), gated(a.gate != nullptr) {}
    template <typename F>
    __device__ void ahead(int n, F fetch) {         // the next n rows' copies; empty groups behind the last row
        for (int i = 0; i < n; ++i) {
            if (fetched < hi) fetch(fetched, fetch_slot);
            feed_commit();
            ++fetched;
            fetch_slot = fetch_slot + 1 == slots ? 0 : fetch_slot + 1;
        }
    }
    // the rows at hand are row .. row + count - 1; true where they begin another group
    __device__ bool next() {
        bool fresh = false;
        if (gated && (group < 0 || row >= group_end)) {
            group = row / group_rows;
            group_end = (group + 1) * group_rows;
            fresh = true;
        }
        const long long end = gated && group_end < hi ? group_end : hi;
        count = end - row < R ? (int)(end - row) : R;
        return fresh;
    }
    __device__ int slot_of(int i) const { const int s = slot + i; return s >= slots ? s - slots : s; }
    __device__ void done() { row += count; slot = slot_of(count); }
};

__device__ __forceinline__ size_t param_bytes(int code) { return code == GB_F32 ? 4 : 2; }

// Mean (0 for rms) and 1 / deviation of R rows.  The variance is that of the centred values, which
// are at hand: a second reduction instead of a difference of large numbers.
template <bool LAYER, int VEC, int NV, int R>
__device__ void row_stats(const Lane<VEC, NV>& lane, float2 (&v)[R][Lane<VEC, NV>::P], float inv_d, float eps,
                          Reducer& reduce, float (&mean)[R], float (&rstd)[R]) {
    constexpr int P = Lane<VEC, NV>::P;
    if constexpr (LAYER) {
        #pragma unroll
        for (int i = 0; i < R; ++i) {
            float2 s = v[i][0];
            #pragma unroll
            for (int e = 1; e < P; ++e) s = add2(s, v[i][e]);
            mean[i] = s.x + s.y;
        }
        reduce.sum(mean);
        #pragma unroll
        for (int i = 0; i < R; ++i) {
            mean[i] *= inv_d;
            #pragma unroll
            for (int e = 0; e < P; ++e) v[i][e] = add2(v[i][e], both(-mean[i]));
            lane.mask(v[i]);
        }
    }
    #pragma unroll
    for (int i = 0; i < R; ++i) {
        float2 q = mul2(v[i][0], v[i][0]);
        #pragma unroll
        for (int e = 1; e < P; ++e) q = fma2(v[i][e], v[i][e], q);
        rstd[i] = q.x + q.y;
    }
    reduce.sum(rstd);
    #pragma unroll
    for (int i = 0; i < R; ++i) rstd[i] = 1.0f / sqrtf(rstd[i] * inv_d + eps);
}

extern __shared__ __align__(16) char join_shared[];

// FULL: layer norms, or any bias; otherwise rms norms without.
template <typename TS, typename TU, typename TY, int VEC, int NV, int R, bool FULL>
__global__ void __launch_bounds__(MAX_THREADS) join_fwd_kernel(const JoinArgs a) {
    __shared__ __align__(16) float buffer[2 * MAX_WARPS * 4];
    using L = Lane<VEC, NV>;
    constexpr int P = L::P;
    const L lane(a.d);
    Feed<TS, VEC, NV> from_residual;
    Feed<TU, VEC, NV> from_update;
    constexpr int BYTES = Feed<TS, VEC, NV>::BYTES + Feed<TU, VEC, NV>::BYTES;
    const uint32_t shared = (uint32_t)__cvta_generic_to_shared(join_shared), per_slot = BYTES * blockDim.x;
    from_residual.place(a.residual, a.residual_stride, shared);
    from_update.place(a.update, a.update_stride, shared + Feed<TS, VEC, NV>::BYTES * blockDim.x);
    Walk<R> walk(a);
    auto fetch = [&](long long row, int slot) {
        from_residual.fetch(lane, row, slot * per_slot);
        from_update.fetch(lane, row, slot * per_slot);
    };
    walk.ahead(walk.slots, fetch);
    Reducer reduce(buffer);
    const float inv_d = 1.0f / (float)a.d;
    float2 w[P], b[P], pw[P], pb[P], gate[P];
    lane.param(a.weight, a.param_code, 1.0f, w);
    lane.param(a.post_weight, a.param_code, 1.0f, pw);
    if (FULL) {
        lane.param(a.bias, a.param_code, 0.0f, b);
        lane.param(a.post_bias, a.param_code, 0.0f, pb);
    }
    lane.fill(a.scale, gate);
    while (walk.row < walk.hi) {
        if (walk.next()) {
            lane.param(static_cast<const char*>(a.gate) + walk.group * a.d * param_bytes(a.gate_code), a.gate_code,
                       1.0f, gate);
            #pragma unroll
            for (int e = 0; e < P; ++e) gate[e] = mul2(gate[e], both(a.scale));
        }
        feed_wait(walk.slots - R);
        float2 u[R][P], r[R][P];
        #pragma unroll
        for (int i = 0; i < R; ++i) {
            if (i < walk.count) {
                const uint32_t at = walk.slot_of(i) * per_slot;
                from_update.get(lane, walk.row + i, at, u[i]);
                from_residual.get(lane, walk.row + i, at, r[i]);
            } else {
                lane.fill(0.0f, u[i]);
                lane.fill(0.0f, r[i]);
            }
        }
        walk.ahead(walk.count, fetch);
        float mean[R] = {}, rstd[R], post_mean[R] = {}, post_rstd[R];
        #pragma unroll
        for (int i = 0; i < R; ++i) rstd[i] = post_rstd[i] = 1.0f;
        if (a.post_weight) {
            if (FULL && a.layer) row_stats<true>(lane, u, inv_d, a.eps, reduce, post_mean, post_rstd);
            else row_stats<false>(lane, u, inv_d, a.eps, reduce, post_mean, post_rstd);
            #pragma unroll
            for (int i = 0; i < R; ++i) {
                #pragma unroll
                for (int e = 0; e < P; ++e) {
                    u[i][e] = mul2(u[i][e], both(post_rstd[i]));
                    u[i][e] = FULL ? fma2(u[i][e], pw[e], pb[e]) : mul2(u[i][e], pw[e]);
                }
            }
        }
        #pragma unroll
        for (int i = 0; i < R; ++i) {
            #pragma unroll
            for (int e = 0; e < P; ++e) {
                r[i][e] = fma2(gate[e], u[i][e], r[i][e]);
                if (sizeof(TS) != 4) {       // the norm that follows is that of the stream as it is stored
                    r[i][e].x = gb_up(gb_down<TS>(r[i][e].x));
                    r[i][e].y = gb_up(gb_down<TS>(r[i][e].y));
                }
            }
            if (FULL) lane.mask(r[i]);
            if (i < walk.count) lane.store(static_cast<TS*>(a.stream) + (walk.row + i) * a.d, r[i]);
        }
        if (a.next) {
            if (FULL && a.layer) row_stats<true>(lane, r, inv_d, a.eps, reduce, mean, rstd);
            else row_stats<false>(lane, r, inv_d, a.eps, reduce, mean, rstd);
            #pragma unroll
            for (int i = 0; i < R; ++i) {
                #pragma unroll
                for (int e = 0; e < P; ++e) {
                    r[i][e] = mul2(r[i][e], both(rstd[i]));
                    r[i][e] = FULL ? fma2(r[i][e], w[e], b[e]) : mul2(r[i][e], w[e]);
                }
                if (i < walk.count) lane.store(static_cast<TY*>(a.normed) + (walk.row + i) * a.d, r[i]);
            }
        }
        if (a.stats && threadIdx.x == 0) {
            #pragma unroll
            for (int i = 0; i < R; ++i)
                if (i < walk.count) a.stats[walk.row + i] = make_float4(post_mean[i], post_rstd[i], mean[i], rstd[i]);
        }
        walk.done();
    }
}

// The sums over R rows that norm' needs: of g x^, and in a layer norm of g.
template <bool FULL, int P, int R>
__device__ void backward_sums(const float2 (&g)[R][P], const float2 (&hat)[R][P], int layer, float inv_d,
                              Reducer& reduce, float (&m1)[R], float (&m0)[R]) {
    #pragma unroll
    for (int i = 0; i < R; ++i) {
        float2 s = mul2(g[i][0], hat[i][0]);
        #pragma unroll
        for (int e = 1; e < P; ++e) s = fma2(g[i][e], hat[i][e], s);
        m1[i] = s.x + s.y;
        m0[i] = 0.0f;
    }
    if (FULL && layer) {
        float all[2 * R];
        #pragma unroll
        for (int i = 0; i < R; ++i) {
            float2 s = g[i][0];
            #pragma unroll
            for (int e = 1; e < P; ++e) s = add2(s, g[i][e]);
            all[2 * i] = m1[i];
            all[2 * i + 1] = s.x + s.y;
        }
        reduce.sum(all);
        #pragma unroll
        for (int i = 0; i < R; ++i) { m1[i] = all[2 * i]; m0[i] = all[2 * i + 1] * inv_d; }
    } else reduce.sum(m1);
    #pragma unroll
    for (int i = 0; i < R; ++i) m1[i] *= inv_d;
}

// One block is one worker.  part[worker] holds, one behind the other, the sums of d_weight,
// d_bias, d_post_weight, d_post_bias that exist.  Worker c and gate group g meet in slot c + g of
// gate_part: along the rows one of the two grows by one at a time, so no two pairs share a slot.
// NEXT: the following norm's gradient takes part; OWN: the update has a norm or a gate of its own.
template <typename TS, typename TU, typename TY, int VEC, int NV, int R, bool FULL, bool NEXT, bool OWN>
__global__ void __launch_bounds__(MAX_THREADS) join_bwd_kernel(const JoinArgs a) {
    __shared__ __align__(16) float buffer[2 * MAX_WARPS * 4];
    using L = Lane<VEC, NV>;
    constexpr int P = L::P;
    const L lane(a.d);
    using FS = Feed<TS, VEC, NV>;
    using FU = Feed<TU, VEC, NV>;
    using FY = Feed<TY, VEC, NV>;
    FS from_grad, from_stream;
    FU from_update;
    FY from_normed;
    constexpr int BYTES = FS::BYTES + (NEXT ? FS::BYTES + FY::BYTES : 0) + (OWN ? FU::BYTES : 0);
    const uint32_t per_slot = BYTES * blockDim.x;
    uint32_t region = (uint32_t)__cvta_generic_to_shared(join_shared);
    from_grad.place(a.d_stream, a.d, region);
    region += FS::BYTES * blockDim.x;
    if (NEXT) {
        from_stream.place(a.stream, a.d, region);
        region += FS::BYTES * blockDim.x;
        from_normed.place(a.d_normed, a.d, region);
        region += FY::BYTES * blockDim.x;
    }
    if (OWN) from_update.place(a.update, a.update_stride, region);
    Walk<R> walk(a);
    auto fetch = [&](long long row, int slot) {
        const uint32_t at = slot * per_slot;
        if (a.d_stream) from_grad.fetch(lane, row, at);
        if (NEXT) {
            from_stream.fetch(lane, row, at);
            from_normed.fetch(lane, row, at);
        }
        if (OWN) from_update.fetch(lane, row, at);
    };
    walk.ahead(walk.slots, fetch);
    Reducer reduce(buffer);
    const float inv_d = 1.0f / (float)a.d;
    float2 w[P], pw[P], pb[P], gate[P];
    float2 dw[P], db[P], dpw[P], dpb[P], dg[P];
    lane.param(a.weight, a.param_code, 1.0f, w);
    lane.param(a.post_weight, a.param_code, 1.0f, pw);
    lane.fill(a.scale, gate);
    lane.fill(0.0f, dw);
    lane.fill(0.0f, dpw);
    lane.fill(0.0f, dg);
    if (FULL) {
        lane.param(a.post_bias, a.param_code, 0.0f, pb);
        lane.fill(0.0f, db);
        lane.fill(0.0f, dpb);
    }
    // d_gate is gathered without the scale, which is put on where it is stored
    auto flush = [&](long long group) {
        #pragma unroll
        for (int e = 0; e < P; ++e) dg[e] = mul2(dg[e], both(a.scale));
        lane.store(a.gate_part + (blockIdx.x + group) * a.d, dg);
        lane.fill(0.0f, dg);
    };
    while (walk.row < walk.hi) {
        const long long before = walk.group;
        const bool fresh = walk.next();
        if (OWN && fresh) {
            if (before >= 0) flush(before);
            lane.param(static_cast<const char*>(a.gate) + walk.group * a.d * param_bytes(a.gate_code), a.gate_code,
                       1.0f, gate);
            #pragma unroll
            for (int e = 0; e < P; ++e) gate[e] = mul2(gate[e], both(a.scale));
        }
        float4 st[R];
        #pragma unroll
        for (int i = 0; i < R; ++i) st[i] = i < walk.count ? a.stats[walk.row + i] : make_float4(0.f, 0.f, 0.f, 0.f);
        feed_wait(walk.slots - R);
        float2 dr[R][P], u[R][P];
        #pragma unroll
        for (int i = 0; i < R; ++i) {
            lane.fill(0.0f, dr[i]);
            if (i < walk.count && a.d_stream) from_grad.get(lane, walk.row + i, walk.slot_of(i) * per_slot, dr[i]);
        }
        if (NEXT) {
            float2 g[R][P], hat[R][P];
            float m1[R], m0[R];
            #pragma unroll
            for (int i = 0; i < R; ++i) {
                lane.fill(0.0f, g[i]);
                lane.fill(0.0f, hat[i]);
                if (i < walk.count) {
                    const uint32_t at = walk.slot_of(i) * per_slot;
                    from_normed.get(lane, walk.row + i, at, g[i]);
                    from_stream.get(lane, walk.row + i, at, hat[i]);
                }
            }
            if (!OWN) walk.ahead(walk.count, fetch);
            #pragma unroll
            for (int i = 0; i < R; ++i) {
                if (FULL && a.layer) {
                    #pragma unroll
                    for (int e = 0; e < P; ++e) hat[i][e] = add2(hat[i][e], both(-st[i].z));
                    lane.mask(hat[i]);
                }
                #pragma unroll
                for (int e = 0; e < P; ++e) {
                    hat[i][e] = mul2(hat[i][e], both(st[i].w));
                    dw[e] = fma2(g[i][e], hat[i][e], dw[e]);
                    if (FULL) db[e] = add2(db[e], g[i][e]);
                    g[i][e] = mul2(g[i][e], w[e]);
                }
            }
            backward_sums<FULL>(g, hat, a.layer, inv_d, reduce, m1, m0);
            #pragma unroll
            for (int i = 0; i < R; ++i) {
                const float2 rs = both(st[i].w), back = both(-m1[i] * st[i].w);
                #pragma unroll
                for (int e = 0; e < P; ++e) {
                    if (FULL) g[i][e] = add2(g[i][e], both(-m0[i]));
                    dr[i][e] = fma2(g[i][e], rs, fma2(hat[i][e], back, dr[i][e]));
                }
                if (FULL) lane.mask(dr[i]);
            }
        }
        if (OWN) {
            #pragma unroll
            for (int i = 0; i < R; ++i) {
                lane.fill(0.0f, u[i]);
                if (i < walk.count) from_update.get(lane, walk.row + i, walk.slot_of(i) * per_slot, u[i]);
            }
        }
        if (OWN || !NEXT) walk.ahead(walk.count, fetch);
        if (a.d_residual) {
            #pragma unroll
            for (int i = 0; i < R; ++i)
                if (i < walk.count) lane.store(static_cast<TS*>(a.d_residual) + (walk.row + i) * a.d, dr[i]);
        }
        if (OWN) {
            #pragma unroll
            for (int i = 0; i < R; ++i) {
                if (FULL && a.layer && a.post_weight) {
                    #pragma unroll
                    for (int e = 0; e < P; ++e) u[i][e] = add2(u[i][e], both(-st[i].x));
                    lane.mask(u[i]);
                }
                #pragma unroll
                for (int e = 0; e < P; ++e) {
                    u[i][e] = mul2(u[i][e], both(st[i].y));            // the update itself without a post norm
                    const float2 v = FULL ? fma2(u[i][e], pw[e], pb[e]) : mul2(u[i][e], pw[e]);
                    dg[e] = fma2(dr[i][e], v, dg[e]);
                    dr[i][e] = mul2(dr[i][e], gate[e]);
                    dpw[e] = fma2(dr[i][e], u[i][e], dpw[e]);
                    if (FULL) dpb[e] = add2(dpb[e], dr[i][e]);
                    dr[i][e] = mul2(dr[i][e], pw[e]);
                }
            }
            if (a.post_weight) {
                float m1[R], m0[R];
                backward_sums<FULL>(dr, u, a.layer, inv_d, reduce, m1, m0);
                #pragma unroll
                for (int i = 0; i < R; ++i) {
                    #pragma unroll
                    for (int e = 0; e < P; ++e) {
                        if (FULL) dr[i][e] = add2(dr[i][e], both(-m0[i]));
                        dr[i][e] = mul2(both(st[i].y), fma2(u[i][e], both(-m1[i]), dr[i][e]));
                    }
                }
            }
        } else {
            #pragma unroll
            for (int i = 0; i < R; ++i) {
                #pragma unroll
                for (int e = 0; e < P; ++e) dr[i][e] = mul2(dr[i][e], gate[e]);
            }
        }
        #pragma unroll
        for (int i = 0; i < R; ++i)
            if (i < walk.count) lane.store(static_cast<TU*>(a.d_update) + (walk.row + i) * a.d, dr[i]);
        walk.done();
    }
    if (OWN && a.gate && walk.group >= 0) flush(walk.group);
    const int sums = (NEXT ? (a.bias ? 2 : 1) : 0) + (a.post_weight ? (a.post_bias ? 2 : 1) : 0);
    float* mine = a.part + (size_t)blockIdx.x * sums * a.d;
    if (NEXT) { lane.store(mine, dw); mine += a.d; }
    if (FULL && NEXT && a.bias) { lane.store(mine, db); mine += a.d; }
    if (OWN && a.post_weight) { lane.store(mine, dpw); mine += a.d; }
    if (FULL && OWN && a.post_weight && a.post_bias) lane.store(mine, dpb);
}

struct SumArgs {
    const float* part;
    const float* gate_part;
    void* out[4];                      // one for each sum, in the order of part
    void* gate_out;                    // [groups][d]
    long long rows, group_rows, groups, workers;
    int d, sums, param_code, gate_code;
};

// Column sums of the partial results: 32 columns a block, SLICES threads share a column, four
// partial results under way in each.
constexpr int SLICES = 32;
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
    if (col < a.d) {
        long long c = lo + threadIdx.y;
        for (; c + 3 * SLICES < hi; c += 4 * SLICES) {
            float v[4];
            #pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = base[(c + i * SLICES) * stride + col];
            #pragma unroll
            for (int i = 0; i < 4; ++i) acc += v[i];
        }
        for (; c < hi; c += SLICES) acc += base[c * stride + col];
    }
    __shared__ float slice[SLICES][33];
    slice[threadIdx.y][threadIdx.x] = acc;
    __syncthreads();
    // warp y sums column y of the block
    const float total = gb_warp_sum(slice[threadIdx.x][threadIdx.y]);
    const int mine = blockIdx.y * 32 + threadIdx.y;
    if (threadIdx.x == 0 && mine < a.d) {
        if (which < a.sums) gb_write(a.out[which], a.param_code, mine, total);
        else gb_write(a.gate_out, a.gate_code, (size_t)(which - a.sums) * a.d + mine, total);
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

// Slots that fit beside one another in an SM's 227 KB.
int slots_for(int bytes_per_slot, int blocks, int rows_at_once) {
    int n = bytes_per_slot ? (int)((220 << 10) / blocks / bytes_per_slot) : MAX_SLOTS;
    return n < rows_at_once ? rows_at_once : n > MAX_SLOTS ? MAX_SLOTS : n;
}

template <typename K>
int start(K kernel, int grid, int threads, int bytes_per_slot, int blocks, int rows_at_once, JoinArgs a, cudaStream_t s) {
    a.slots = slots_for(bytes_per_slot, blocks, rows_at_once);
    const int shared = a.slots * bytes_per_slot;
    if (shared > (40 << 10)) {                       // more than a launch may take unasked, with the static part
        const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared);
        if (err != cudaSuccess) return (int)err;
    }
    kernel<<<grid, threads, shared, s>>>(a);
    return (int)cudaGetLastError();
}

template <typename TS, typename TU, typename TY, int VEC, int NV, int R, bool FULL>
int launch_form(bool forward, int threads, const JoinArgs& a, cudaStream_t s) {
    constexpr int S = Feed<TS, VEC, NV>::BYTES, U = Feed<TU, VEC, NV>::BYTES, Y = Feed<TY, VEC, NV>::BYTES;
    const int blocks = blocks_per_sm(threads);
    const int grid = workers_for(a.rows, threads);
    if (forward) return start(join_fwd_kernel<TS, TU, TY, VEC, NV, R, FULL>, grid, threads, (S + U) * threads, blocks, R, a, s);
    const bool next = a.d_normed, own = a.post_weight || a.gate;
    if (next && own) return start(join_bwd_kernel<TS, TU, TY, VEC, NV, R, FULL, true, true>, grid, threads, (2 * S + Y + U) * threads, blocks, R, a, s);
    if (next) return start(join_bwd_kernel<TS, TU, TY, VEC, NV, R, FULL, true, false>, grid, threads, (2 * S + Y) * threads, blocks, R, a, s);
    return start(join_bwd_kernel<TS, TU, TY, VEC, NV, R, FULL, false, true>, grid, threads, (S + U) * threads, blocks, R, a, s);
}

template <typename TS, typename TU, typename TY, int VEC, int NV, int R>
int launch_shaped(bool forward, int threads, const JoinArgs& a, cudaStream_t s) {
    if (a.layer || a.bias || a.post_bias) return launch_form<TS, TU, TY, VEC, NV, R, true>(forward, threads, a, s);
    return launch_form<TS, TU, TY, VEC, NV, R, false>(forward, threads, a, s);
}

template <typename TS, typename TU, typename TY>
int launch(bool forward, int vec, const JoinArgs& a, cudaStream_t s) {
    const Shape shape = shape_of(a.d, vec);
    if (vec == 8) {
        if (shape.rounds == 1) return launch_shaped<TS, TU, TY, 8, 1, 2>(forward, shape.threads, a, s);
        return launch_shaped<TS, TU, TY, 8, 2, 1>(forward, shape.threads, a, s);
    }
    if (shape.rounds <= 1) return launch_shaped<TS, TU, TY, 1, 1, 2>(forward, shape.threads, a, s);
    if (shape.rounds <= 4) return launch_shaped<TS, TU, TY, 1, 4, 2>(forward, shape.threads, a, s);
    return launch_shaped<TS, TU, TY, 1, 16, 1>(forward, shape.threads, a, s);
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
