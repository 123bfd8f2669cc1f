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
// both gradients, the stream and the update and writes two gradients.  A row belongs to a team of
// threads, 16 or 24 columns each; its values stay in registers between the reductions while the
// next rows are already on their way to shared memory.  A team walks several rows, so that the
// gradients of the parameters, sums over all rows, are gathered in registers; a block leaves its
// teams' sums and a second launch adds the blocks' in index order.
//
// One B200, forward / backward with the sums, launches included (an empty launch is 2.6 us):
//   8192 x 768, layer norm, fp32 stream and bf16 update     22 / 26 us   (75 / 113 MB: 12 / 18 us)
//   8192 x 2048, bf16, both norms and a gate                 29 / 43 us   (134 / 201 MB: 21 / 31 us)
//   4096 x 4096, bf16, both norms and sequence gates         31 / 55 us   (the same bytes)
//   3333 x 1001, fp32, post norm and sequence gates          18 / 25 us   (40 / 53 MB: 6 / 8 us)
// What it took at 8192 x 2048: loads in registers and one barrier after another 186 us; rows staged
// ahead 132; packed arithmetic and two rows at a time 99; 16 columns a thread instead, with copies
// that need no branch, 94; parameters in shared memory instead of spilled registers 77; sums of one
// block an SM added by wide loads 73.  Odd widths move single values, and the widest rows have few
// warps to hide a row's two reductions: there it is instructions that bind.
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
    float* part;                       // [blocks][sums][d]
    float* gate_part;                  // [owners + groups - 1][d]
    long long rows, group_rows;        // rows of one gate group
    int d, layer, param_code, gate_code, next, slots;
    int owners;                        // teams that have rows, at least one each
    float scale, eps;
};

constexpr int MAX_THREADS = 512;
constexpr int REDUCER_FLOATS = 2 * 2 * (MAX_THREADS / 32) * 4;   // two to four warps a team take the room of four

// A block is blockDim.y teams of blockDim.x threads; a team owns a row.  An SM holds one block, so
// that a backward pass leaves one row of partial sums for each SM.
__device__ __forceinline__ int team_of_grid() { return blockIdx.x * blockDim.y + threadIdx.y; }

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

// Sums of Q values over a team's threads, one barrier a reduction: the buffers alternate.  Within
// a warp two values are exchanged for one another before they are added: five shuffles for either.
struct Reducer {
    float* buffer;                     // [2][warps, to a multiple of four][4]
    int warps, half, parity;
    __device__ explicit Reducer(float* b) : warps((int)blockDim.x >> 5), half((warps + 3) / 4 * 16), parity(0) {
        buffer = b + threadIdx.y * 2 * half;
        if (warps == 1) return;
        for (int i = threadIdx.x; i < 2 * half; i += blockDim.x) buffer[i] = 0.0f;
        team_barrier();
    }
    __device__ static void team_barrier() {
        asm volatile("bar.sync %0, %1;" :: "r"((int)threadIdx.y + 1), "r"((int)blockDim.x) : "memory");
    }
    template <int Q>
    __device__ void sum(float (&v)[Q]) {
        static_assert(Q == 1 || Q == 2, "values of one reduction");
        const int lane = threadIdx.x & 31;
        float mine = v[0];
        if constexpr (Q == 2) {
            const bool upper = lane & 16;
            mine = upper ? v[1] : v[0];
            mine += __shfl_xor_sync(0xffffffffu, upper ? v[0] : v[1], 16);
        }
        #pragma unroll
        for (int step = Q == 2 ? 8 : 16; step > 0; step >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, step);
        if (warps == 1) {
            #pragma unroll
            for (int q = 0; q < Q; ++q) v[q] = Q == 1 ? mine : __shfl_sync(0xffffffffu, mine, q * (32 / Q));
            return;
        }
        float* b = buffer + parity * half;
        parity ^= 1;
        if (lane % (32 / Q) == 0) b[(threadIdx.x >> 5) * Q + lane / (32 / Q)] = mine;
        team_barrier();
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

// Two values rounded to T, as floats.
template <typename T> __device__ __forceinline__ float2 rounded(float2 v) { return v; }
template <> __device__ __forceinline__ float2 rounded<__nv_bfloat16>(float2 v) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
    const uint32_t w = reinterpret_cast<const uint32_t&>(h);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 rounded<__half>(float2 v) {
    return __half22float2(__floats2half2_rn(v.x, v.y));
}

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
    template <bool WIDE = false>
    __device__ void param(const void* p, int code, float otherwise, float2 (&v)[P]) const {
        fill(otherwise, v);
        if (!p) return;
        if (code == GB_F32) read<WIDE>(static_cast<const float*>(p), v);
        else if (code == GB_BF16) read<WIDE>(static_cast<const __nv_bfloat16*>(p), v);
        else read<WIDE>(static_cast<const __half*>(p), v);
    }
    template <bool WIDE, typename T>
    __device__ void read(const T* p, float2 (&v)[P]) const {
        if constexpr (VEC == 8 && WIDE) {
            if (reinterpret_cast<uintptr_t>(p) % (8 * sizeof(T)) == 0) {
                Raw8<T> raw[NV];
                #pragma unroll
                for (int k = 0; k < NV; ++k) if (ok[k]) raw[k].load(p + col[k]);
                #pragma unroll
                for (int k = 0; k < NV; ++k) {
                    if (!ok[k]) continue;
                    float f[8];
                    raw[k].get(f);
                    #pragma unroll
                    for (int j = 0; j < 8; ++j) at(v, k * 8 + j) = f[j];
                }
                return;
            }
        }
        #pragma unroll
        for (int e = 0; e < E; ++e) if (ok[e / VEC]) at(v, e) = gb_up(p[col[e / VEC] + e % VEC]);
    }
};

// Rows of one tensor on their way to this thread's registers.  Each thread copies the values that
// it will use itself into its own places in shared memory (cp.async), as many rows ahead as there
// are slots, so the loads of several rows are in flight while a row is reduced, no register holds
// them and no barrier guards them.  A copy of no bytes fills its place with zeros and reads
// nothing: so it is for columns and rows that do not exist.  Single values of two bytes cannot be
// copied so: they are read when used.
template <typename T, int VEC, int NV>
struct Feed {
    static constexpr bool STAGED = VEC == 8 || sizeof(T) == 4;
    static constexpr int PIECE = VEC == 8 ? 16 : 4;                     // bytes of one copy
    static constexpr int PIECES = VEC == 8 ? (int)sizeof(T) / 2 : 1;    // copies a vector
    static constexpr int BYTES = STAGED ? NV * PIECES * PIECE : 0;      // a thread and slot
    using L = Lane<VEC, NV>;
    const char* ahead;                 // this thread's first value of the next row to fetch
    const char* here;                  // of the row at hand, where rows are not staged
    long long step;                    // bytes from row to row
    uint32_t place;                    // of this thread's first piece in a slot
    __device__ void open(const void* p, long long row_stride, long long row, uint32_t region) {
        step = row_stride * (long long)sizeof(T);
        ahead = here = static_cast<const char*>(p) + row * step + threadIdx.x * (VEC * (int)sizeof(T));
        place = region + threadIdx.x * PIECE;
    }
    __device__ void fetch(const L& lane, uint32_t slot, bool exists) {
        if constexpr (STAGED) {
            #pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int bytes = exists && lane.ok[k] ? PIECE : 0;
                #pragma unroll
                for (int h = 0; h < PIECES; ++h) {
                    const uint32_t to = place + slot + (k * PIECES + h) * (int)blockDim.x * PIECE;
                    const char* from = ahead + (long long)(k * (int)blockDim.x * (VEC * (int)sizeof(T)) + h * 16);
                    if constexpr (PIECE == 16)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(to), "l"(from), "r"(bytes) : "memory");
                    else
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" :: "r"(to), "l"(from), "r"(bytes) : "memory");
                }
            }
            ahead += step;
        }
    }
    __device__ void get(const L& lane, uint32_t slot, float2 (&v)[L::P]) {
        if (L::E & 1) v[L::P - 1].y = 0.0f;
        #pragma unroll
        for (int k = 0; k < NV; ++k) {
            if constexpr (VEC == 8) {
                float f[8];
                #pragma unroll
                for (int h = 0; h < PIECES; ++h) {
                    uint4 q;
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                                 : "r"(place + slot + (k * PIECES + h) * (int)blockDim.x * PIECE) : "memory");
                    if constexpr (sizeof(T) == 4) {
                        f[4 * h] = __uint_as_float(q.x); f[4 * h + 1] = __uint_as_float(q.y);
                        f[4 * h + 2] = __uint_as_float(q.z); f[4 * h + 3] = __uint_as_float(q.w);
                    } else {
                        Raw8<T> raw;
                        raw.q = q;
                        raw.get(f);
                    }
                }
                #pragma unroll
                for (int j = 0; j < 8; ++j) L::at(v, k * 8 + j) = f[j];
            } else if constexpr (STAGED) {
                float f;
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(place + slot + k * (int)blockDim.x * PIECE) : "memory");
                L::at(v, k) = f;
            } else {
                const T* row = reinterpret_cast<const T*>(here);
                L::at(v, k) = lane.ok[k] ? gb_up(row[k * (int)blockDim.x]) : 0.0f;
            }
        }
        if constexpr (!STAGED) here += step;
    }
};

// Rows of a result, one behind the other.
template <typename T, int VEC, int NV>
struct Sink {
    using L = Lane<VEC, NV>;
    T* at;
    __device__ void open(void* p, long long row, int d) { at = static_cast<T*>(p) + row * d + threadIdx.x * VEC; }
    __device__ void put(const L& lane, const float2 (&v)[L::P], int d) {
        #pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (!lane.ok[k]) continue;
            if constexpr (VEC == 8) {
                float f[8];
                #pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = L::at(v, k * 8 + j);
                gb_store8(at + k * (int)blockDim.x * 8, f);
            } else at[k * (int)blockDim.x] = gb_down<T>(L::at(v, k));
        }
        at += d;
    }
};

__device__ __forceinline__ void feed_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// waits until at most `behind` of the groups this thread committed are under way
__device__ __forceinline__ void feed_wait(int behind) {
    switch (behind) {
        case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
        case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
        case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
        default: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
    }
}
constexpr int MAX_SLOTS = 4;

// Worker (team) c owns the rows [first_row(c), first_row(c + 1)); owner_of is its inverse.
__host__ __device__ __forceinline__ long long first_row(long long c, long long rows, long long workers) {
    return c * rows / workers;
}
__host__ __device__ __forceinline__ long long owner_of(long long row, long long rows, long long workers) {
    return ((row + 1) * workers - 1) / rows;
}

__device__ __forceinline__ size_t param_bytes(int code) { return code == GB_F32 ? 4 : 2; }

// A parameter's values in a thread's columns, as fp32: in registers, or in the thread's own places
// in shared memory, where the sums of the backward pass need the registers (8192 x 2048 with both
// norms and a gate: spilled registers cost more than the reads).
template <int VEC, int NV, bool SHARED>
struct Held {
    using L = Lane<VEC, NV>;
    static constexpr int PIECE = VEC == 8 ? 16 : 4;
    static constexpr int BYTES = SHARED ? L::E * 4 : 0;       // a thread
    float2 v[SHARED ? 1 : L::P];
    uint32_t place;
    __device__ void set(const float2 (&x)[L::P], uint32_t region) {
        place = region + threadIdx.x * PIECE;
        if constexpr (!SHARED) {
            #pragma unroll
            for (int e = 0; e < L::P; ++e) v[e] = x[e];
        } else if constexpr (VEC == 8) {
            #pragma unroll
            for (int i = 0; i < L::E / 4; ++i)
                asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};"
                             :: "r"(place + i * (int)blockDim.x * 16), "f"(x[2 * i].x), "f"(x[2 * i].y),
                                "f"(x[2 * i + 1].x), "f"(x[2 * i + 1].y) : "memory");
        } else {
            #pragma unroll
            for (int e = 0; e < L::E; ++e)
                asm volatile("st.shared.f32 [%0], %1;" :: "r"(place + e * (int)blockDim.x * 4), "f"(L::at(x, e)) : "memory");
        }
    }
    __device__ void get(float2 (&x)[L::P]) const {
        if constexpr (!SHARED) {
            #pragma unroll
            for (int e = 0; e < L::P; ++e) x[e] = v[e];
        } else if constexpr (VEC == 8) {
            #pragma unroll
            for (int i = 0; i < L::E / 4; ++i)
                asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(x[2 * i].x), "=f"(x[2 * i].y), "=f"(x[2 * i + 1].x), "=f"(x[2 * i + 1].y)
                             : "r"(place + i * (int)blockDim.x * 16) : "memory");
        } else {
            if (L::E & 1) x[L::P - 1].y = 0.0f;
            #pragma unroll
            for (int e = 0; e < L::E; ++e)
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(L::at(x, e)) : "r"(place + e * (int)blockDim.x * 4) : "memory");
        }
    }
};

// The scale times the gate of the row at hand, read where a row begins another group.
template <int VEC, int NV, bool SHARED>
struct Gate {
    using L = Lane<VEC, NV>;
    Held<VEC, NV, SHARED> held;
    long long group = -1, end;
    uint32_t region;
    __device__ Gate(const JoinArgs& a, long long lo, uint32_t region_) : end(a.gate ? lo : a.rows), region(region_) {
        float2 v[L::P];
        L::fill(a.scale, v);
        held.set(v, region);
    }
    __device__ void move(const JoinArgs& a, const L& lane, long long row) {
        group = row / a.group_rows;
        end = (group + 1) * a.group_rows;
        float2 v[L::P];
        lane.param(static_cast<const char*>(a.gate) + group * a.d * param_bytes(a.gate_code), a.gate_code, 1.0f, v);
        #pragma unroll
        for (int e = 0; e < L::P; ++e) v[e] = mul2(v[e], both(a.scale));
        held.set(v, region);
    }
};

// Mean (0 for rms) and 1 / deviation of a row, which is centred in place.  The variance is that of
// the centred values: a second reduction instead of a difference of large numbers.
template <bool FULL, int VEC, int NV>
__device__ float2 row_stats(const Lane<VEC, NV>& lane, float2 (&v)[Lane<VEC, NV>::P], int layer, float inv_d,
                            float eps, Reducer& reduce) {
    constexpr int P = Lane<VEC, NV>::P;
    float mean = 0.0f;
    if (FULL && layer) {
        float2 s = v[0];
        #pragma unroll
        for (int e = 1; e < P; ++e) s = add2(s, v[e]);
        float sum[1] = {s.x + s.y};
        reduce.sum(sum);
        mean = sum[0] * inv_d;
        #pragma unroll
        for (int e = 0; e < P; ++e) v[e] = add2(v[e], both(-mean));
        lane.mask(v);
    }
    float2 q = mul2(v[0], v[0]);
    #pragma unroll
    for (int e = 1; e < P; ++e) q = fma2(v[e], v[e], q);
    float sum[1] = {q.x + q.y};
    reduce.sum(sum);
    return make_float2(mean, rsqrtf(sum[0] * inv_d + eps));          // 2 ulp
}

extern __shared__ __align__(16) char join_shared[];

// FULL: layer norms, or any bias; otherwise rms norms without.
// OWN: the update has a norm or a gate of its own.
template <int VEC, int NV, bool FULL, bool OWN> constexpr bool FORWARD_SHARED = FULL && OWN && VEC * NV > 8 && NV < 16;
template <typename TS, typename TU, typename TY, int VEC, int NV, bool FULL, bool OWN>
__global__ void __launch_bounds__(NV == 3 ? 384 : MAX_THREADS) join_fwd_kernel(const JoinArgs a) {
    __shared__ __align__(16) float buffer[REDUCER_FLOATS];
    using L = Lane<VEC, NV>;
    constexpr int P = L::P;
    if (team_of_grid() >= a.owners) return;          // a team's barriers are its own
    const L lane(a.d);
    const long long lo = first_row(team_of_grid(), a.rows, a.owners), hi = first_row(team_of_grid() + 1LL, a.rows, a.owners);
    constexpr bool SHARED = FORWARD_SHARED<VEC, NV, FULL, OWN>;
    using H = Held<VEC, NV, SHARED>;
    const uint32_t per_slot = (Feed<TS, VEC, NV>::BYTES + Feed<TU, VEC, NV>::BYTES) * blockDim.x;
    const uint32_t held_bytes = H::BYTES * blockDim.x;
    // the teams' columns are the same: they share the parameters, and each has its gate and slots
    const uint32_t held_at = (uint32_t)__cvta_generic_to_shared(join_shared);
    const uint32_t gate_at = held_at + 4 * held_bytes + threadIdx.y * (a.slots * per_slot + held_bytes);
    const uint32_t mine = gate_at + held_bytes;
    Feed<TS, VEC, NV> from_residual;
    Feed<TU, VEC, NV> from_update;
    from_residual.open(a.residual, a.residual_stride, lo, mine);
    from_update.open(a.update, a.update_stride, lo, mine + Feed<TS, VEC, NV>::BYTES * blockDim.x);
    for (int i = 0; i < a.slots; ++i) {
        from_update.fetch(lane, i * per_slot, lo + i < hi);
        from_residual.fetch(lane, i * per_slot, lo + i < hi);
        feed_commit();
    }
    Sink<TS, VEC, NV> to_stream;
    Sink<TY, VEC, NV> to_normed;
    to_stream.open(a.stream, lo, a.d);
    to_normed.open(a.normed, lo, a.d);
    Reducer reduce(buffer);
    const float inv_d = 1.0f / (float)a.d;
    H weight, bias, post_weight, post_bias;
    auto hold = [&](H& held, const void* p, float otherwise, int i) {
        float2 v[P];
        lane.template param<true>(p, a.param_code, otherwise, v);
        held.set(v, held_at + i * held_bytes);
    };
    hold(weight, a.weight, 1.0f, 0);
    if (FULL) hold(bias, a.bias, 0.0f, 1);
    if (OWN) hold(post_weight, a.post_weight, 1.0f, 2);
    if (OWN && FULL) hold(post_bias, a.post_bias, 0.0f, 3);
    Gate<VEC, NV, SHARED> gate(a, lo, gate_at);
    uint32_t slot = 0;
    const uint32_t last_slot = (a.slots - 1) * per_slot;
    for (long long row = lo; row < hi; ++row) {
        if (OWN && row >= gate.end) gate.move(a, lane, row);
        feed_wait(a.slots - 1);
        float2 u[P], r[P];
        from_update.get(lane, slot, u);
        from_residual.get(lane, slot, r);
        from_update.fetch(lane, slot, row + a.slots < hi);
        from_residual.fetch(lane, slot, row + a.slots < hi);
        feed_commit();
        slot = slot == last_slot ? 0 : slot + per_slot;
        float2 post = make_float2(0.0f, 1.0f), next = make_float2(0.0f, 1.0f);
        if (OWN && a.post_weight) {
            post = row_stats<FULL>(lane, u, a.layer, inv_d, a.eps, reduce);
            float2 pw[P], pb[P];
            post_weight.get(pw);
            if (FULL) post_bias.get(pb);
            #pragma unroll
            for (int e = 0; e < P; ++e) {
                u[e] = mul2(u[e], both(post.y));
                u[e] = FULL ? fma2(u[e], pw[e], pb[e]) : mul2(u[e], pw[e]);
            }
        }
        {
            float2 g[P];
            if (OWN) gate.held.get(g);
            else lane.fill(a.scale, g);
            #pragma unroll
            for (int e = 0; e < P; ++e)          // the norm that follows is that of the stream as it is stored
                r[e] = rounded<TS>(fma2(g[e], u[e], r[e]));
        }
        to_stream.put(lane, r, a.d);
        if (a.next) {
            if (FULL) lane.mask(r);
            next = row_stats<FULL>(lane, r, a.layer, inv_d, a.eps, reduce);
            float2 w[P], b[P];
            weight.get(w);
            if (FULL) bias.get(b);
            #pragma unroll
            for (int e = 0; e < P; ++e) {
                r[e] = mul2(r[e], both(next.y));
                r[e] = FULL ? fma2(r[e], w[e], b[e]) : mul2(r[e], w[e]);
            }
            to_normed.put(lane, r, a.d);
        }
        if (a.stats && threadIdx.x == 0) a.stats[row] = make_float4(post.x, post.y, next.x, next.y);
    }
}

// The means over a row that norm' needs: of g x^, and in a layer norm of g.
template <bool FULL, int P>
__device__ float2 backward_means(const float2 (&g)[P], const float2 (&hat)[P], int layer, float inv_d, Reducer& reduce) {
    float2 s = mul2(g[0], hat[0]);
    #pragma unroll
    for (int e = 1; e < P; ++e) s = fma2(g[e], hat[e], s);
    if (FULL && layer) {
        float2 z = g[0];
        #pragma unroll
        for (int e = 1; e < P; ++e) z = add2(z, g[e]);
        float two[2] = {s.x + s.y, z.x + z.y};
        reduce.sum(two);
        return make_float2(two[0] * inv_d, two[1] * inv_d);
    }
    float one[1] = {s.x + s.y};
    reduce.sum(one);
    return make_float2(one[0] * inv_d, 0.0f);
}

// part[block] holds, one behind the other, the sums of d_weight, d_bias, d_post_weight, d_post_bias
// that exist; the teams of a block add theirs up first.  Team c and gate group g meet in slot c + g
// of gate_part: along the rows one of the two grows by one at a time, so no two pairs share a slot.
// MOST: threads of the largest block, which sets the registers that a thread may have.
// NEXT: the following norm's gradient takes part; OWN: the update has a norm or a gate of its own.
// SHARED: the parameters are held in shared memory.
template <typename TS, typename TU, typename TY, int VEC, int NV, int MOST, bool SHARED, bool FULL, bool NEXT, bool OWN>
__global__ void __launch_bounds__(MOST) join_bwd_kernel(const JoinArgs a) {
    __shared__ __align__(16) float buffer[REDUCER_FLOATS];
    using L = Lane<VEC, NV>;
    constexpr int P = L::P;
    const L lane(a.d);
    const bool owner = team_of_grid() < a.owners;
    const long long lo = owner ? first_row(team_of_grid(), a.rows, a.owners) : 0;
    const long long hi = owner ? first_row(team_of_grid() + 1LL, a.rows, a.owners) : 0;
    using FS = Feed<TS, VEC, NV>;
    using FU = Feed<TU, VEC, NV>;
    using FY = Feed<TY, VEC, NV>;
    FS from_grad, from_stream;
    FU from_update;
    FY from_normed;
    const uint32_t per_slot = (FS::BYTES + (NEXT ? FS::BYTES + FY::BYTES : 0) + (OWN ? FU::BYTES : 0)) * blockDim.x;
    using H = Held<VEC, NV, SHARED>;
    const uint32_t held_bytes = H::BYTES * blockDim.x;
    constexpr int HELD = (NEXT ? 1 : 0) + (OWN ? (FULL ? 2 : 1) : 0);
    // the teams' columns are the same: they share the parameters, and each has its gate and slots
    uint32_t held_at = (uint32_t)__cvta_generic_to_shared(join_shared);
    const uint32_t gate_at = held_at + HELD * held_bytes + threadIdx.y * (a.slots * per_slot + (OWN ? held_bytes : 0));
    uint32_t region = gate_at + (OWN ? held_bytes : 0);
    from_grad.open(a.d_stream, a.d, lo, region);
    region += FS::BYTES * blockDim.x;
    if (NEXT) {
        from_stream.open(a.stream, a.d, lo, region);
        region += FS::BYTES * blockDim.x;
        from_normed.open(a.d_normed, a.d, lo, region);
        region += FY::BYTES * blockDim.x;
    }
    if (OWN) from_update.open(a.update, a.update_stride, lo, region);
    auto fetch = [&](uint32_t at, bool exists) {
        if (NEXT) {
            from_normed.fetch(lane, at, exists);
            from_stream.fetch(lane, at, exists);
        }
        from_grad.fetch(lane, at, exists && a.d_stream);
        if (OWN) from_update.fetch(lane, at, exists && (a.post_weight || a.gate));
        feed_commit();
    };
    for (int i = 0; i < a.slots; ++i) fetch(i * per_slot, lo + i < hi);
    Sink<TS, VEC, NV> to_residual;
    Sink<TU, VEC, NV> to_update;
    to_residual.open(a.d_residual, lo, a.d);
    to_update.open(a.d_update, lo, a.d);
    Reducer reduce(buffer);
    const float inv_d = 1.0f / (float)a.d;
    Gate<VEC, NV, SHARED && OWN> gate(a, lo, gate_at);
    H weight, post_weight, post_bias;
    auto hold = [&](H& held, const void* p, float otherwise) {
        float2 v[P];
        lane.template param<true>(p, a.param_code, otherwise, v);
        held.set(v, held_at);
        held_at += held_bytes;
    };
    if (NEXT) hold(weight, a.weight, 1.0f);
    if (OWN) hold(post_weight, a.post_weight, 1.0f);
    if (OWN && FULL) hold(post_bias, a.post_bias, 0.0f);
    float2 dw[P], db[P], dpw[P], dpb[P], dg[P];
    lane.fill(0.0f, dw);
    lane.fill(0.0f, dpw);
    lane.fill(0.0f, dg);
    lane.fill(0.0f, db);
    lane.fill(0.0f, dpb);
    auto flush = [&]() {                 // d_gate is gathered without the scale
        #pragma unroll
        for (int e = 0; e < P; ++e) dg[e] = mul2(dg[e], both(a.scale));
        lane.store(a.gate_part + (team_of_grid() + gate.group) * a.d, dg);
        lane.fill(0.0f, dg);
    };
    uint32_t slot = 0;
    const uint32_t last_slot = (a.slots - 1) * per_slot;
    float4 coming = lo < hi ? a.stats[lo] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (long long row = lo; row < hi; ++row) {
        if (OWN && row >= gate.end) {
            if (gate.group >= 0) flush();
            gate.move(a, lane, row);
        }
        const float4 st = coming;
        if (row + 1 < hi) coming = a.stats[row + 1];
        feed_wait(a.slots - 1);
        float2 dr[P], u[P];
        if (NEXT) {
            float2 g[P], hat[P];
            from_normed.get(lane, slot, g);
            from_stream.get(lane, slot, hat);
            if (FULL && a.layer) {
                #pragma unroll
                for (int e = 0; e < P; ++e) hat[e] = add2(hat[e], both(-st.z));
                lane.mask(hat);
            }
            float2 w[P];
            weight.get(w);
            #pragma unroll
            for (int e = 0; e < P; ++e) {
                hat[e] = mul2(hat[e], both(st.w));
                dw[e] = fma2(g[e], hat[e], dw[e]);
                if (FULL) db[e] = add2(db[e], g[e]);
                g[e] = mul2(g[e], w[e]);
            }
            const float2 m = backward_means<FULL>(g, hat, a.layer, inv_d, reduce);
            if (a.d_stream) from_grad.get(lane, slot, dr);
            else lane.fill(0.0f, dr);
            const float2 r = both(st.w), back = both(-m.x * st.w);
            #pragma unroll
            for (int e = 0; e < P; ++e) {
                if (FULL) g[e] = add2(g[e], both(-m.y));
                dr[e] = fma2(g[e], r, fma2(hat[e], back, dr[e]));
            }
            if (FULL) lane.mask(dr);
        } else from_grad.get(lane, slot, dr);        // without a following norm there is a gradient here
        if (OWN) from_update.get(lane, slot, u);
        fetch(slot, row + a.slots < hi);
        slot = slot == last_slot ? 0 : slot + per_slot;
        if (a.d_residual) to_residual.put(lane, dr, a.d);
        if (OWN) {
            if (FULL && a.layer && a.post_weight) {
                #pragma unroll
                for (int e = 0; e < P; ++e) u[e] = add2(u[e], both(-st.x));
                lane.mask(u);
            }
            float2 pw[P], pb[P], gv[P];
            post_weight.get(pw);
            if (FULL) post_bias.get(pb);
            gate.held.get(gv);
            #pragma unroll
            for (int e = 0; e < P; ++e) {
                u[e] = mul2(u[e], both(st.y));            // the update itself without a post norm
                const float2 v = FULL ? fma2(u[e], pw[e], pb[e]) : mul2(u[e], pw[e]);
                dg[e] = fma2(dr[e], v, dg[e]);
                dr[e] = mul2(dr[e], gv[e]);
                dpw[e] = fma2(dr[e], u[e], dpw[e]);
                if (FULL) dpb[e] = add2(dpb[e], dr[e]);
                dr[e] = mul2(dr[e], pw[e]);
            }
            if (a.post_weight) {
                const float2 m = backward_means<FULL>(dr, u, a.layer, inv_d, reduce);
                #pragma unroll
                for (int e = 0; e < P; ++e) {
                    if (FULL) dr[e] = add2(dr[e], both(-m.y));
                    dr[e] = mul2(both(st.y), fma2(u[e], both(-m.x), dr[e]));
                }
            }
        } else {
            #pragma unroll
            for (int e = 0; e < P; ++e) dr[e] = mul2(dr[e], both(a.scale));
        }
        if (a.d_update) to_update.put(lane, dr, a.d);
    }
    if (OWN && a.gate && gate.group >= 0) flush();
    const int sums = (NEXT ? (a.bias ? 2 : 1) : 0) + (a.post_weight ? (a.post_bias ? 2 : 1) : 0);
    float* mine = a.part + (size_t)blockIdx.x * sums * a.d;
    auto leave = [&](const float2 (&v)[P]) {
        if (blockDim.y == 1) lane.store(mine, v);
        else {                          // the slots are free now: a team's row of d floats each
            const uint32_t at = (uint32_t)__cvta_generic_to_shared(join_shared);
            __syncthreads();
            Held<VEC, NV, true> place;          // thread by thread, as it is read below
            place.set(v, at + threadIdx.y * place.BYTES * blockDim.x);
            __syncthreads();
            if (threadIdx.y == 0) {
                float2 total[P], more[P];
                #pragma unroll
                for (int e = 0; e < P; ++e) total[e] = v[e];
                for (int y = 1; y < blockDim.y; ++y) {
                    place.place = at + y * place.BYTES * blockDim.x + threadIdx.x * place.PIECE;
                    place.get(more);
                    #pragma unroll
                    for (int e = 0; e < P; ++e) total[e] = add2(total[e], more[e]);
                }
                lane.store(mine, total);
            }
        }
        mine += a.d;
    };
    if (blockDim.y > 1) asm volatile("cp.async.wait_all;" ::: "memory");
    if (NEXT) leave(dw);
    if (FULL && NEXT && a.bias) leave(db);
    if (OWN && a.post_weight) leave(dpw);
    if (FULL && OWN && a.post_weight && a.post_bias) leave(dpb);
}

struct SumArgs {
    const float* part;
    const float* gate_part;
    void* out[4];                      // one for each sum, in the order of part
    void* gate_out;                    // [groups][d]
    long long rows, group_rows, groups;
    int blocks, owners;                // rows of part, teams that own rows
    int d, sums, param_code, gate_code;
};

// Column sums of the partial results: a block takes 32 columns, W at a load, and its threads share
// their partial rows, of which there is one an SM.
template <int W>
__global__ void __launch_bounds__(256) join_sum_kernel(const SumArgs a) {
    constexpr int ACROSS = 32 / W, SLICES = 256 / ACROSS;
    const int x = threadIdx.x % ACROSS, y = threadIdx.x / ACROSS;
    const int col = blockIdx.y * 32 + x * W;
    const long long which = blockIdx.x;
    const float* base;
    int lo = 0, hi = a.blocks;
    size_t stride;
    if (which < a.sums) {
        base = a.part + which * a.d;
        stride = (size_t)a.sums * a.d;
    } else {
        const long long g = which - a.sums;
        if (a.groups == 1) hi = a.owners;
        else {
            lo = (int)owner_of(g * a.group_rows, a.rows, a.owners);
            hi = (int)owner_of((g + 1) * a.group_rows - 1, a.rows, a.owners) + 1;
        }
        base = a.gate_part + g * a.d;
        stride = a.d;
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");           // the partial results are there
    float acc[W];
    #pragma unroll
    for (int j = 0; j < W; ++j) acc[j] = 0.0f;
    if (col < a.d) {
        const float* from = base + (size_t)(lo + y) * stride + col;
        #pragma unroll 4
        for (int c = lo + y; c < hi; c += SLICES, from += SLICES * stride) {
            if constexpr (W == 4) {
                const float4 v = *reinterpret_cast<const float4*>(from);
                acc[0] += v.x; acc[1] += v.y; acc[2] += v.z; acc[3] += v.w;
            } else acc[0] += *from;
        }
    }
    __shared__ float slice[SLICES][33];
    #pragma unroll
    for (int j = 0; j < W; ++j) slice[y][x * W + j] = acc[j];
    __syncthreads();
    // eight threads a column, each an eighth of its slices
    const int mine = threadIdx.x / 8, part = threadIdx.x % 8;
    float total = 0.0f;
    #pragma unroll
    for (int s = part; s < SLICES; s += 8) total += slice[s][mine];
    #pragma unroll
    for (int o = 4; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const int out = blockIdx.y * 32 + mine;
    if (part == 0 && out < a.d) {
        if (which < a.sums) gb_write(a.out[which], a.param_code, out, total);
        else gb_write(a.gate_out, a.gate_code, (size_t)(which - a.sums) * a.d + out, total);
    }
}

constexpr int MAX_WIDTH = 8192;

// How rows of d values in vectors of vec are dealt out: threads of a team, teams of a block, rounds
// of vectors a thread.  Eight columns a thread up to 256, then 16 or 24: what a row costs beside
// its values (addresses, the reduction) is shared by more of them.  Up to 768 columns a row is a
// warp's, without a barrier.  Single values: four a thread, and up to sixteen where that is more
// threads than a block may have.
// A block has as many teams as its registers allow (128 a thread forward, 168 backward up to 4096
// columns), fewer where there are not rows enough for every SM.
struct Shape { int threads, teams, rounds; };
Shape shape_of(long long rows, int d, int vec, bool forward) {
    const int vectors = (d + vec - 1) / vec;
    Shape s{0, 1, 1};
    if (vec == 8) {
        s.rounds = vectors <= 96 ? (vectors + 31) / 32 : 2;
        s.threads = vectors <= 96 ? 32 : ((vectors + 1) / 2 + 31) / 32 * 32;
    } else {
        const int most = vectors > 1024 ? MAX_THREADS : 256;
        s.threads = ((vectors + 3) / 4 + 31) / 32 * 32;
        if (s.threads > most) s.threads = most;
        s.rounds = (vectors + s.threads - 1) / s.threads;
    }
    const int most = (forward && s.rounds != 3) || s.threads > 384 ? 512 : 384;
    const long long enough = (rows + 147) / 148;
    s.teams = most / s.threads;
    if (s.teams > 15) s.teams = 15;                  // a barrier each, and one for all
    if (s.teams > enough) s.teams = (int)enough;
    if (s.teams < 1) s.teams = 1;
    return s;
}
int blocks_for(long long rows, const Shape& s) {
    const long long want = (rows + s.teams - 1) / s.teams;
    return (int)(want < 148 ? want : 148);
}
int owners_for(long long rows, const Shape& s) {
    const long long teams = (long long)blocks_for(rows, s) * s.teams;
    return (int)(rows < teams ? rows : teams);
}

constexpr int MAX_SHARED = 225 << 10;

// A launch with as many slots as fit in an SM.  `common` bytes a thread are the teams' together,
// `own` each team's, beside `slot` for every slot.
template <typename K>
int start(K kernel, const Shape& shape, int slot, int common, int own, int add, JoinArgs a, cudaStream_t s) {
    const int room = (MAX_SHARED - common * shape.threads) / shape.teams - own * shape.threads;
    a.slots = slot ? room / (slot * shape.threads) : MAX_SLOTS;
    if (a.slots > MAX_SLOTS) a.slots = MAX_SLOTS;
    if (a.slots < 1) a.slots = 1;
    int shared = ((a.slots * slot + own) * shape.teams + common) * shape.threads;
    const int sums = shape.teams > 1 ? shape.teams * add * shape.threads : 0;          // where the teams add up
    if (shared < sums) shared = sums;
    if (shared > (40 << 10)) {                       // more than a launch may take unasked, with the static part
        const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared);
        if (err != cudaSuccess) return (int)err;
    }
    a.owners = owners_for(a.rows, shape);
    kernel<<<blocks_for(a.rows, shape), dim3(shape.threads, shape.teams), shared, s>>>(a);
    return (int)cudaGetLastError();
}

template <typename TS, typename TU, typename TY, int VEC, int NV, int MOST, bool FULL, bool SHARED>
int launch_backward(const Shape& shape, const JoinArgs& a, cudaStream_t s) {
    constexpr int S = Feed<TS, VEC, NV>::BYTES, U = Feed<TU, VEC, NV>::BYTES, Y = Feed<TY, VEC, NV>::BYTES;
    constexpr int H = Held<VEC, NV, SHARED>::BYTES, A = Held<VEC, NV, true>::BYTES, O = FULL ? 2 : 1;
    const bool next = a.d_normed, own = a.post_weight || a.gate;
    if (next && own) return start(join_bwd_kernel<TS, TU, TY, VEC, NV, MOST, SHARED, FULL, true, true>, shape, 2 * S + Y + U, (1 + O) * H, H, A, a, s);
    if (next) return start(join_bwd_kernel<TS, TU, TY, VEC, NV, MOST, SHARED, FULL, true, false>, shape, 2 * S + Y, H, 0, A, a, s);
    return start(join_bwd_kernel<TS, TU, TY, VEC, NV, MOST, SHARED, FULL, false, true>, shape, S + U, O * H, H, A, a, s);
}

template <typename TS, typename TU, typename TY, int VEC, int NV, int MOST, bool FULL>
int launch_form(bool forward, const Shape& shape, const JoinArgs& a, cudaStream_t s) {
    constexpr int S = Feed<TS, VEC, NV>::BYTES, U = Feed<TU, VEC, NV>::BYTES, Y = Feed<TY, VEC, NV>::BYTES;
    if (forward) {
        constexpr int H = Held<VEC, NV, FORWARD_SHARED<VEC, NV, FULL, true>>::BYTES;
        if (a.post_weight || a.gate)
            return start(join_fwd_kernel<TS, TU, TY, VEC, NV, FULL, true>, shape, S + U, 4 * H, H, 0, a, s);
        return start(join_fwd_kernel<TS, TU, TY, VEC, NV, FULL, false>, shape, S + U, 0, 0, 0, a, s);
    }
    // the widest rows of fp32 with four parameters leave no room for a slot: registers hold those
    if constexpr (MOST == 512 && FULL && sizeof(TU) == 4) {
        constexpr int H = Held<VEC, NV, true>::BYTES;
        if ((4 * H + 2 * S + Y + U) * shape.threads > MAX_SHARED)
            return launch_backward<TS, TU, TY, VEC, NV, MOST, FULL, false>(shape, a, s);
    }
    return launch_backward<TS, TU, TY, VEC, NV, MOST, FULL, true>(shape, a, s);
}

template <typename TS, typename TU, typename TY, int VEC, int NV, int MOST>
int launch_shaped(bool forward, const Shape& shape, const JoinArgs& a, cudaStream_t s) {
    if (a.layer || a.bias || a.post_bias) return launch_form<TS, TU, TY, VEC, NV, MOST, true>(forward, shape, a, s);
    return launch_form<TS, TU, TY, VEC, NV, MOST, false>(forward, shape, a, s);
}

template <typename TS, typename TU, typename TY>
int launch(bool forward, int vec, const JoinArgs& a, cudaStream_t s) {
    const Shape shape = shape_of(a.rows, a.d, vec, forward);
    if (vec == 8) {
        if (shape.rounds == 1) return launch_shaped<TS, TU, TY, 8, 1, 384>(forward, shape, a, s);
        if (shape.rounds == 3) return launch_shaped<TS, TU, TY, 8, 3, 384>(forward, shape, a, s);
        if (shape.threads * shape.teams <= 384) return launch_shaped<TS, TU, TY, 8, 2, 384>(forward, shape, a, s);
        return launch_shaped<TS, TU, TY, 8, 2, 512>(forward, shape, a, s);
    }
    if (shape.rounds <= 4 && (forward || shape.threads <= 384)) return launch_shaped<TS, TU, TY, 1, 4, 384>(forward, shape, a, s);
    return launch_shaped<TS, TU, TY, 1, 16, 512>(forward, shape, a, s);
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

// Blocks of a backward call and teams of them that own rows: part holds blocks * sums * d floats,
// gate_part (owners + groups - 1) * d.
extern "C" void gb_residual_norm_workers(long long rows, int d, int vec, int* blocks, int* owners) {
    const Shape s = shape_of(rows, d, vec, false);
    *blocks = blocks_for(rows, s);
    *owners = owners_for(rows, s);
}

// The stream, both gradients (either may be null) and the outputs are [rows, d] without gaps;
// d_residual and d_update may be null.  out: the gradients of weight, bias, post_weight, post_bias that exist
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
    gb_residual_norm_workers(rows, d, vec, &q.blocks, &q.owners);
    q.d = d; q.param_code = param_code; q.gate_code = gate_code;
    q.sums = (d_normed ? (bias ? 2 : 1) : 0) + (post_weight ? (post_bias ? 2 : 1) : 0);
    const long long what = q.sums + q.groups;
    if (what == 0) return 0;
    if (what > 0x7fffffff) return (int)cudaErrorInvalidValue;
    // its blocks may be set up while the last of the gradients are on their way
    cudaLaunchAttribute overlap = {};
    overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    overlap.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)what, (d + 31) / 32);
    config.blockDim = dim3(256);
    config.stream = cuda_stream;
    config.attrs = &overlap;
    config.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&config, d % 4 ? join_sum_kernel<1> : join_sum_kernel<4>, q);
}
