// block_norm.cu -- the norms around a block of a residual stack fused with the block's
// gate and the residual scale, forward and backward, fp32 math.
//
//   r1 = rsqrt(mean(y^2) + eps)      u = y r1 gamma_post        (u = y without gamma_post)
//   h' = alpha h + gate u
//   r2 = rsqrt(mean(h'^2) + eps)     x = h' r2 gamma_pre
//
// Backward, from y and the stored h' (D columns, rows independent but for the sums):
//   g2 = dx gamma_pre, n2 = h' r2    dt = dh' + r2 (g2 - n2 mean(g2 n2))
//   dh = alpha dt, du = gate dt      dgate = sum dt u, dgamma_pre = sum dx n2
//   g1 = du gamma_post, n1 = y r1    dy = r1 (g1 - n1 mean(g1 n1)), dgamma_post = sum du n1
//
// Bound by HBM: every row of y, h (and dx, dh') is read once and every result
// written once; a row stays in registers between its two reductions.  A thread owns
// 8 consecutive columns (one 16-byte piece of a bf16 row).  Rows of at most 256 columns
// belong to one warp (shuffles only), wider ones to a CTA.  16384 rows of 2048: forward with
// a bf16 stream 46.1 us (268 MB, 5.8 TB/s), backward with an fp32 stream 117 us (604 MB,
// 5.2 TB/s; 7 us of it the column sums); 8 rows of 2048 forward 2.4 us.  Above 4096 columns the
// backward's 1024 threads have 64 registers each, the whole register file, for values that take
// 125: they spill, and 8192 columns run at 2.3 TB/s with an fp32 stream (1.7 with bf16, where the
// spills weigh more), against 5.3 at 4096.
#include "common.cuh"

namespace gdn {
namespace {

constexpr int kNarrow = 256;          // widest row that one warp holds, 8 columns a lane
constexpr int kNarrowRows = 8;        // rows (warps) per CTA then
constexpr int kMaxD = 8192;           // 1024 threads x 8 columns

struct BlockNormArgs {
    const uint16_t* y;
    const void* h;                    // forward: h; backward: the stored h'
    const uint16_t* gamma_post;
    const uint16_t* gate;
    const uint16_t* gamma_pre;
    void* h_out;                      // backward: dh
    uint16_t* x;                      // backward: dy
    const void* dh_out;
    const uint16_t* dx;
    unsigned int* err;                // backward
    float alpha, eps;
    int R, D;
    int rows_per_gate;                // rows that share a gate row (R: one gate row for all)
};

__device__ __forceinline__ void unpack8(const uint4& w, float (&f)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(u[i] << 16);
        f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}
// Eight consecutive values of a row as loaded: bf16 stays packed until it is used.
template <bool F32>
struct Piece {
    uint4 w[F32 ? 2 : 1];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (F32 ? 2 : 1); ++i) w[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void load(const void* base, long at) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) + at * (F32 ? 4 : 2));
#pragma unroll
        for (int i = 0; i < (F32 ? 2 : 1); ++i) w[i] = __ldcg(p + i);
    }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                f[4 * i] = __uint_as_float(w[i].x);
                f[4 * i + 1] = __uint_as_float(w[i].y);
                f[4 * i + 2] = __uint_as_float(w[i].z);
                f[4 * i + 3] = __uint_as_float(w[i].w);
            }
        } else {
            unpack8(w[0], f);
        }
    }
};
template <bool F32>
__device__ __forceinline__ void store8(void* base, long at, const float (&f)[8]) {
    if constexpr (F32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + at);
        p[0] = make_float4(f[0], f[1], f[2], f[3]);
        p[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at) =
            make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
    }
}
// a weight's eight values, 1 without it
__device__ __forceinline__ void weight8(const uint16_t* p, long at, bool on, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 1.f;
    if (on && p) unpack8(__ldg(reinterpret_cast<const uint4*>(p + at)), f);
}

// Sum over the row's threads: one warp, or the whole CTA through `red` ([2][32] floats,
// used in turn so that one barrier per sum is enough).
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float* red, int& turn) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (!WARP) {
        float* mine = red + turn * 32;
        turn ^= 1;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
        if (lane == 0) mine[warp] = v;
        __syncthreads();
        v = lane < nw ? mine[lane] : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}

// A CTA walks over rows with the weights in registers (a gate row too, where all rows
// share it) and the next row's loads in flight while it works on one.
template <bool F32, bool WARP, int NT>
__global__ void __launch_bounds__(NT, NT == 256 ? 4 : 1) block_norm_fwd_kernel(const BlockNormArgs a) {
    __shared__ float red[2][32];
    pdl_launch_dependents();
    const int piece = WARP ? (threadIdx.x & 31) : threadIdx.x, col = piece * 8;
    const bool on = col < a.D;
    const long row0 = WARP ? static_cast<long>(blockIdx.x) * kNarrowRows + (threadIdx.x >> 5) : blockIdx.x;
    const long step = WARP ? static_cast<long>(gridDim.x) * kNarrowRows : gridDim.x;
    const float inv_d = 1.f / static_cast<float>(a.D);
    const bool one_gate = a.gate && a.rows_per_gate == a.R, row_gate = a.gate && !one_gate;
    float wp[8], wq[8];                        // gamma_post (times the gate that all rows share), gamma_pre
    weight8(a.gamma_post, col, on, wp);
    weight8(a.gamma_pre, col, on, wq);
    pdl_wait_prior();                          // y, h and the gate (an activation too) come from earlier kernels
    if (one_gate && on) {
        float g[8];
        unpack8(__ldcg(reinterpret_cast<const uint4*>(a.gate + col)), g);
#pragma unroll
        for (int i = 0; i < 8; ++i) wp[i] *= g[i];
    }
    Piece<false> ny, ng;
    Piece<F32> nh;
    ny.zero();
    nh.zero();
    ng.zero();
    auto fetch = [&](long r) {
        if (!on || r >= a.R) return;
        ny.load(a.y, r * a.D + col);
        nh.load(a.h, r * a.D + col);
        if (row_gate) ng.load(a.gate, (r / a.rows_per_gate) * a.D + col);
    };
    fetch(row0);
    int turn = 0;
    for (long r = row0; r < a.R; r += step) {
        const long at = r * a.D + col;
        float u[8], h[8], g[8];
        ny.get(u);
        nh.get(h);
        ng.get(g);
        fetch(r + step);
        float r1 = 1.f;
        if (a.gamma_post) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += u[i] * u[i];
            r1 = rsqrtf(row_sum<WARP>(ss, &red[0][0], turn) * inv_d + a.eps);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] *= r1 * wp[i];
        if (row_gate)
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] *= g[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = fmaf(a.alpha, h[i], u[i]);
        if (on) store8<F32>(a.h_out, at, h);
        if (a.gamma_pre) {
            float ss = 0.f;
            if (on)
#pragma unroll
                for (int i = 0; i < 8; ++i) ss += h[i] * h[i];
            const float r2 = rsqrtf(row_sum<WARP>(ss, &red[0][0], turn) * inv_d + a.eps);
            if (on) {
#pragma unroll
                for (int i = 0; i < 8; ++i) h[i] *= r2 * wq[i];
                store8<false>(a.x, at, h);
            }
        }
    }
}

// The rows a backward work item covers: every parts-th row of one gate row's rows, so the
// column sums of an item belong to one gate row.  CTAs side by side take rows side by
// side (contiguous shares: 122 us instead of 118 at 16384 x 2048, fp32 stream).
struct BwdPlan {
    int groups;                       // gate rows that are summed over rows (1 when none are)
    int parts;                        // parts per group
    int ctas;
};

// The six sums of a backward row in one round: after three steps of exchanging halves a
// lane holds one of the (eight) values for four lanes, two more steps finish it.
template <bool WARP>
__device__ __forceinline__ void row_sums6(float (&v)[8], float* red, int& turn) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int n = 4, o = 16; n >= 1; n >>= 1, o >>= 1) {
        const bool up = (lane & o) != 0;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float send = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
    }
    float s = v[0];
    s += __shfl_xor_sync(0xffffffffu, s, 2);
    s += __shfl_xor_sync(0xffffffffu, s, 1);
    // value index of a lane: bits 4, 3, 2
    if constexpr (!WARP) {
        float* mine = red + turn * 256;                         // [8 values][32 warps]
        turn ^= 1;
        const int idx = lane >> 2, nw = blockDim.x >> 5;
        if ((lane & 3) == 0) mine[idx * 32 + warp] = s;
        __syncthreads();
        s = 0.f;
        for (int w = lane & 3; w < nw; w += 4) s += mine[idx * 32 + w];
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        s += __shfl_xor_sync(0xffffffffu, s, 1);
    }
#pragma unroll
    for (int i = 0; i < 6; ++i) v[i] = __shfl_sync(0xffffffffu, s, i * 4);
}

__device__ __forceinline__ uint64_t twice(float x) { return pack2(x, x); }
__device__ __forceinline__ void pairs_of(const uint4& w, uint64_t (&p)[4]) {          // 8 bf16
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = pack2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
}
__device__ __forceinline__ uint4 bf16_of(const uint64_t (&p)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float x, y;
        unpack2(p[i], x, y);
        w[i] = pack_bf16x2(x, y);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// eight values of a row in memory (global or shared) as pairs, and back
template <bool F32>
__device__ __forceinline__ void read_pairs(const void* at, uint64_t (&p)[4]) {
    if constexpr (F32) {
        const ulonglong2 a = *static_cast<const ulonglong2*>(at), b = *(static_cast<const ulonglong2*>(at) + 1);
        p[0] = a.x; p[1] = a.y; p[2] = b.x; p[3] = b.y;
    } else {
        pairs_of(*static_cast<const uint4*>(at), p);
    }
}
template <bool F32>
__device__ __forceinline__ void write_pairs(void* base, long at, const uint64_t (&p)[4]) {
    if constexpr (F32) {
        ulonglong2* d = reinterpret_cast<ulonglong2*>(static_cast<float*>(base) + at);
        d[0] = make_ulonglong2(p[0], p[1]);
        d[1] = make_ulonglong2(p[2], p[3]);
    } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at) = bf16_of(p);
    }
}
__device__ __forceinline__ void weight_pairs(const uint16_t* p, long at, bool on, uint64_t (&w)[4]) {
    float f[8];
    weight8(p, at, on, f);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack2(f[2 * i], f[2 * i + 1]);
}

// A backward row and the column sums of the rows before it, eight columns a thread.
// All sums that a row's result needs come before any of it (so one barrier per row): with
// w = gate gamma_post, g2 = dx gamma_pre
//   sum y^2, sum h'^2, A = sum g2 h', B = sum w y dh', C = sum w y g2, E = sum w y h'
//   mean(g2 n2) = r2 A / D,  sum g1 n1 = r1 (B + r2 C - r2^3 (A / D) E)
// Where the rows of an item share their gate row, dgate and dgamma_post both follow from
// q = sum dt n1, so one sum serves both.  Without a norm its input is not looked at (h' is 0
// then, y in dgate only): an infinity there would reach the result as 0 times infinity.
template <bool F32, bool WARP>
struct BwdRow {
    uint64_t gq[4], w[4], q[4], sum_pre[4];    // gamma_pre; gate gamma_post; column sums
    // y, h, dx (both 0 without gamma_pre), dt (dh'): the row's values; gate, sum_post: of a row with a gate row of its own
    template <class AfterSums>
    __device__ __forceinline__ void run(const BlockNormArgs& a, uint64_t (&y)[4], uint64_t (&h)[4], uint64_t (&dx)[4],
                                        uint64_t (&dt)[4], const uint64_t* gate, const uint64_t* gp, uint64_t* sum_post,
                                        void* dgate_rows, int dgate_f32, long at, bool on, float* red, int& turn,
                                        AfterSums after) {
        const float inv_d = 1.f / static_cast<float>(a.D);
        uint64_t t[6] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t x = mul2(dx[i], gq[i]), wy = mul2(w[i], y[i]);
            t[0] = fma2(y[i], y[i], t[0]);
            t[1] = fma2(h[i], h[i], t[1]);
            t[2] = fma2(x, h[i], t[2]);
            t[3] = fma2(wy, dt[i], t[3]);
            t[4] = fma2(wy, x, t[4]);
            t[5] = fma2(wy, h[i], t[5]);
        }
        float s[8];
        s[6] = s[7] = 0.f;
#pragma unroll
        for (int i = 0; i < 6; ++i) {
            float lo, hi;
            unpack2(t[i], lo, hi);
            s[i] = lo + hi;
        }
        row_sums6<WARP>(s, red, turn);
        after();
        const float r1 = a.gamma_post ? rsqrtf(s[0] * inv_d + a.eps) : 1.f;
        const float r2 = a.gamma_pre ? rsqrtf(s[1] * inv_d + a.eps) : 0.f;          // 0: dt = dh'
        const float k = r2 * r2 * r2 * s[2] * inv_d;
        const float m1 = a.gamma_post ? r1 * (s[3] + r2 * s[4] - k * s[5]) * inv_d : 0.f;
        const uint64_t r1_2 = twice(r1), r2_2 = twice(r2), k_2 = twice(-k), m_2 = twice(-m1), al = twice(a.alpha);
        uint64_t out[4], dg[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t n1 = mul2(y[i], r1_2), xr = mul2(dx[i], r2_2);
            sum_pre[i] = fma2(xr, h[i], sum_pre[i]);
            dt[i] = fma2(h[i], k_2, fma2(xr, gq[i], dt[i]));
            out[i] = mul2(al, dt[i]);
            if (gate) {
                const uint64_t e = mul2(dt[i], n1);
                dg[i] = mul2(e, gp[i]);
                sum_post[i] = fma2(e, gate[i], sum_post[i]);
            } else {
                q[i] = fma2(dt[i], n1, q[i]);
            }
            const uint64_t g1 = mul2(dt[i], w[i]);
            y[i] = mul2(r1_2, a.gamma_post ? fma2(n1, m_2, g1) : g1);               // dy
        }
        if (!on) return;
        write_pairs<F32>(a.h_out, at, out);
        write_pairs<false>(a.x, at, y);
        if (gate) {
            if (dgate_f32)
                write_pairs<true>(dgate_rows, at, dg);
            else
                write_pairs<false>(dgate_rows, at, dg);
        }
    }
};

// The walk over items shared by the two backward kernels: dgamma partials [ctas][2][D],
// dgate partials [groups * parts][D]; write_cols(v, dst) adds up and stores a CTA's columns.
template <bool F32, bool WARP, class Rows, class WriteCols>
__device__ __forceinline__ void bwd_items(const BlockNormArgs& a, const BwdPlan& plan, int col, bool on, bool row_gate,
                                          float* part_gamma, float* part_gate, Rows rows, WriteCols write_cols) {
    BwdRow<F32, WARP> st;
    uint64_t sum_post[4] = {};
    weight_pairs(a.gamma_pre, col, on, st.gq);
#pragma unroll
    for (int i = 0; i < 4; ++i) st.sum_pre[i] = 0;
    const int items = plan.groups * plan.parts;
    const long group_rows = a.R / plan.groups;
    for (int it = blockIdx.x; it < items; it += gridDim.x) {
        const int g = it / plan.parts, part = it % plan.parts;
        uint64_t gp[4], gt[4];
        weight_pairs(a.gamma_post, col, on, gp);
        weight_pairs(row_gate ? nullptr : a.gate, static_cast<long>(g) * a.D + col, on, gt);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            st.w[i] = mul2(gp[i], gt[i]);
            st.q[i] = 0;
        }
        rows(st, gp, sum_post, g * group_rows + part, (g + 1) * group_rows, static_cast<long>(plan.parts));
        if (!row_gate) {
            // read again: they are not kept over the rows
            weight_pairs(a.gamma_post, col, on, gp);
            weight_pairs(a.gate, static_cast<long>(g) * a.D + col, on, gt);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sum_post[i] = fma2(st.q[i], gt[i], sum_post[i]);
                st.q[i] = mul2(st.q[i], gp[i]);
            }
            if (part_gate) write_cols(st.q, part_gate + static_cast<long>(it) * a.D);
        }
    }
    if (part_gamma) {
        write_cols(sum_post, part_gamma + (static_cast<long>(blockIdx.x) * 2) * a.D);
        write_cols(st.sum_pre, part_gamma + (static_cast<long>(blockIdx.x) * 2 + 1) * a.D);
    }
}

// Narrow rows: a warp each.
template <bool F32>
__global__ void __launch_bounds__(32 * kNarrowRows, 2)
block_norm_bwd_narrow_kernel(const BlockNormArgs a, const BwdPlan plan, void* dgate_rows, int dgate_f32, float* part_gamma,
                             float* part_gate) {
    extern __shared__ float cols[];                             // [rows of the CTA][D] for the column sums
    const int sub = threadIdx.x >> 5, col = (threadIdx.x & 31) * 8;
    const bool on = col < a.D, row_gate = dgate_rows != nullptr;
    pdl_launch_dependents();
    auto rows = [&](BwdRow<F32, true>& st, const uint64_t (&gp)[4], uint64_t (&sum_post)[4], long r0, long r1, long step) {
        int turn = 0;
        for (long r = r0 + sub * step; r < r1; r += kNarrowRows * step) {
            const long at = r * a.D + col;
            uint64_t y[4] = {}, h[4] = {}, dx[4] = {}, dt[4] = {}, gt[4] = {};
            if (on) {
                read_pairs<false>(a.y + at, y);
                if (a.gamma_pre) {
                    read_pairs<F32>(static_cast<const uint8_t*>(a.h) + at * (F32 ? 4 : 2), h);
                    read_pairs<false>(a.dx + at, dx);
                }
                if (a.dh_out) read_pairs<F32>(static_cast<const uint8_t*>(a.dh_out) + at * (F32 ? 4 : 2), dt);
                if (row_gate) {
                    read_pairs<false>(a.gate + at, gt);
#pragma unroll
                    for (int i = 0; i < 4; ++i) st.w[i] = mul2(gp[i], gt[i]);
                }
            }
            st.run(a, y, h, dx, dt, row_gate ? gt : nullptr, gp, sum_post, dgate_rows, dgate_f32, at, on, nullptr, turn, [] {});
        }
    };
    // sum over the CTA's warps of the lanes' columns, in warp order
    auto write_cols = [&](const uint64_t (&v)[4], float* dst) {
        __syncthreads();
        if (on) write_pairs<true>(cols, sub * a.D + col, v);
        __syncthreads();
        for (int c = threadIdx.x; c < a.D; c += blockDim.x) {
            float s = 0.f;
            for (int w = 0; w < kNarrowRows; ++w) s += cols[w * a.D + c];
            dst[c] = s;
        }
    };
    bwd_items<F32, true>(a, plan, col, on, row_gate, part_gamma, part_gate, rows, write_cols);
}

// Wide rows: a CTA each, through a ring of `stages` rows in shared memory that bulk copies
// fill (y, dx, h', dh', gate row), so that several rows are in flight without registers.
// A thread has its row in registers before the barrier of the sums, so behind that barrier the
// stage is free and takes the row `stages` further on.
struct BwdRing {
    int stages, bytes;                // bytes of a stage
    int off_dx, off_h, off_dh, off_gate;
};
constexpr int kMaxStages = 8;

template <bool F32, int NT>
__global__ void __launch_bounds__(NT, NT == 256 ? 2 : 1)
block_norm_bwd_kernel(const BlockNormArgs a, const BwdPlan plan, const BwdRing ring, void* dgate_rows, int dgate_f32,
                      float* part_gamma, float* part_gate) {
    extern __shared__ __align__(128) uint8_t ring_mem[];
    __shared__ float red[2][256];
    __shared__ uint64_t full[kMaxStages];
    __shared__ int dead_flag;
    volatile int* dead = &dead_flag;
    const int tid = threadIdx.x, col = tid * 8;
    const bool on = col < a.D, row_gate = dgate_rows != nullptr;
    if (tid == 0) {
        for (int i = 0; i < ring.stages; ++i) mbar_init(&full[i], 1);
        dead_flag = 0;
        fence_mbar_init();
    }
    pdl_launch_dependents();
    __syncthreads();
    constexpr int HB = F32 ? 4 : 2;
    uint32_t used = 0;                                          // rows taken from the ring so far
    int turn = 0;
    auto issue = [&](long r, uint32_t n) {                      // one thread: row r as the ring's n-th
        uint8_t* s = ring_mem + (n % ring.stages) * ring.bytes;
        uint64_t* bar = &full[n % ring.stages];
        const uint32_t e = a.D;
        const long at = r * a.D;
        mbar_arrive_expect_tx(bar, e * 2 + (a.gamma_pre ? e * (2 + HB) : 0) + (a.dh_out ? e * HB : 0) + (row_gate ? e * 2 : 0));
        bulk_load(s, a.y + at, e * 2, bar);
        if (a.gamma_pre) {
            bulk_load(s + ring.off_h, static_cast<const uint8_t*>(a.h) + at * HB, e * HB, bar);
            bulk_load(s + ring.off_dx, a.dx + at, e * 2, bar);
        }
        if (a.dh_out) bulk_load(s + ring.off_dh, static_cast<const uint8_t*>(a.dh_out) + at * HB, e * HB, bar);
        if (row_gate) bulk_load(s + ring.off_gate, a.gate + at, e * 2, bar);
    };
    auto rows = [&](BwdRow<F32, false>& st, const uint64_t (&gp)[4], uint64_t (&sum_post)[4], long r0, long r1, long step) {
        if (tid == 0) {
            uint32_t n = used;
            for (long r = r0; r < r1 && n < used + ring.stages; r += step) issue(r, n++);
        }
        for (long r = r0; r < r1; r += step, ++used) {
            const long at = r * a.D + col;
            const uint8_t* s = ring_mem + (used % ring.stages) * ring.bytes;
            // gives up with the error word set; the rows then hold anything, the walk ends as usual
            mbar_wait_or_abort(&full[used % ring.stages], (used / ring.stages) & 1u, a.err, dead);
            uint64_t y[4] = {}, h[4] = {}, dx[4] = {}, dt[4] = {}, gt[4] = {};
            if (on) {
                read_pairs<false>(s + col * 2, y);
                if (a.gamma_pre) {
                    read_pairs<F32>(s + ring.off_h + col * HB, h);
                    read_pairs<false>(s + ring.off_dx + col * 2, dx);
                }
                if (a.dh_out) read_pairs<F32>(s + ring.off_dh + col * HB, dt);
                if (row_gate) {
                    read_pairs<false>(s + ring.off_gate + col * 2, gt);
#pragma unroll
                    for (int i = 0; i < 4; ++i) st.w[i] = mul2(gp[i], gt[i]);
                }
            }
            st.run(a, y, h, dx, dt, row_gate ? gt : nullptr, gp, sum_post, dgate_rows, dgate_f32, at, on, &red[0][0], turn, [&] {
                if (tid == 0 && r + ring.stages * step < r1) issue(r + ring.stages * step, used + ring.stages);
            });
        }
    };
    auto write_cols = [&](const uint64_t (&v)[4], float* dst) {
        if (on) write_pairs<true>(dst, col, v);
    };
    bwd_items<F32, false>(a, plan, col, on, row_gate, part_gamma, part_gate, rows, write_cols);
    __syncthreads();
    if (dead_flag && tid == 0)                                  // gave up: let the copies in flight land
        for (uint32_t n = used > static_cast<uint32_t>(ring.stages) ? used - ring.stages : 0; n < used; ++n)
            mbar_wait(&full[n % ring.stages], (n / ring.stages) & 1u, a.err);
}

// out[o][c] = sum over n of in[(o * n_stride_o + n * n_stride)][c]: 32 columns a CTA, each of
// its 16 warps every 16th n (loads in batches of 8), then the warps' sums in order.
struct SumJob {
    const float* in;
    float* out;
    long o_stride, n_stride;          // elements
    int n;
};
constexpr int kSumWarps = 16;
constexpr int kMaxGridY = 65535;        // more gate rows take turns
__global__ void __launch_bounds__(32 * kSumWarps)
column_sum_kernel(const SumJob j0, const SumJob j1, const SumJob j2, int groups, int D) {
    __shared__ float part[kSumWarps][32];
    pdl_wait_prior();
    // blockIdx.y 0: dgamma_post, 1: dgamma_pre, 2 + g: gate row g
    const SumJob& j = blockIdx.y == 0 ? j0 : blockIdx.y == 1 ? j1 : j2;
    if (!j.out) return;
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
    const int end = blockIdx.y < 2 ? 1 : groups, step = blockIdx.y < 2 ? 1 : gridDim.y - 2;
    for (long o = blockIdx.y < 2 ? 0 : blockIdx.y - 2; o < end; o += step) {
        float s = 0.f;
        if (c < D) {
            const float* p = j.in + o * j.o_stride + c;
            for (int n0 = k; n0 < j.n; n0 += 8 * kSumWarps) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = n0 + i * kSumWarps < j.n ? __ldcg(p + (n0 + i * kSumWarps) * j.n_stride) : 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) s += v[i];
            }
        }
        __syncthreads();                                       // `part` has been read
        part[k][threadIdx.x & 31] = s;
        __syncthreads();
        if (k == 0 && c < D) {
#pragma unroll
            for (int i = 1; i < kSumWarps; ++i) s += part[i][threadIdx.x & 31];
            j.out[o * D + c] = s;
        }
    }
}

int block_threads(int D) { return D <= kNarrow ? 32 * kNarrowRows : (D / 8 + 31) / 32 * 32; }

// backward CTAs per SM, at 128 registers a thread
int bwd_resident(int D) { return block_threads(D) < 512 ? 512 / block_threads(D) : 1; }

// `groups`: gate rows whose gradient is a sum over rows (1 without such a sum).
BwdPlan bwd_plan(int R, int D, int groups) {
    BwdPlan p;
    p.groups = groups;
    const int per_cta = D <= kNarrow ? kNarrowRows : 1;
    const int want = 148 * bwd_resident(D);
    const long group_rows = R / groups;
    long parts = (want + groups - 1) / groups;
    if (parts > (group_rows + per_cta - 1) / per_cta) parts = (group_rows + per_cta - 1) / per_cta;
    p.parts = static_cast<int>(parts < 1 ? 1 : parts);
    const long items = static_cast<long>(groups) * p.parts;
    p.ctas = static_cast<int>(items < want ? items : want);
    return p;
}

int check_block_norm(const char* name, const void* y, const void* h, int h_dtype, const void* gamma_post,
                     const void* gate, int gate_rows, const void* gamma_pre, int R, int D) {
    if (!y || !h) return fail(GDN_ERR_NULL, "%s: y and the residual are required", name);
    if (h_dtype != GDN_DTYPE_BF16 && h_dtype != GDN_DTYPE_F32)
        return fail(GDN_ERR_DTYPE, "%s: h_dtype must be GDN_DTYPE_BF16 or GDN_DTYPE_F32", name);
    if (R < 0 || D <= 0 || D % 8 != 0 || D > kMaxD)
        return fail(GDN_ERR_SHAPE, "%s: need R >= 0 and 0 < D <= %d with D %% 8 == 0 (got R=%d D=%d)", name, kMaxD, R, D);
    if (gate && (gate_rows < 1 || (R > 0 && (gate_rows > R || R % gate_rows != 0))))
        return fail(GDN_ERR_SHAPE, "%s: gate_rows=%d must divide R=%d", name, gate_rows, R);
    for (const void* p : {y, h, gamma_post, gate, gamma_pre})
        if (!aligned16(p)) return fail(GDN_ERR_ALIGN, "%s: pointers must be 16-byte aligned", name);
    return GDN_OK;
}

template <bool F32>
int launch_fwd(const BlockNormArgs& a, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = launch_overlap() ? 1 : 0;
    cfg.stream = st;
    const int nt = block_threads(a.D);
    cfg.blockDim = dim3(nt);
    const int rows = a.D <= kNarrow ? kNarrowRows : 1;
    // as many CTAs as are resident at once (48 registers a thread), each for several rows
    const int most = 148 * (1024 / nt > 0 ? 1024 / nt : 1), need = a.R / rows + (a.R % rows != 0);
    cfg.gridDim = dim3(need < most ? need : most);
    cudaError_t e;
    if (a.D <= kNarrow)
        e = cudaLaunchKernelEx(&cfg, block_norm_fwd_kernel<F32, true, 256>, a);
    else if (nt <= 256)
        e = cudaLaunchKernelEx(&cfg, block_norm_fwd_kernel<F32, false, 256>, a);
    else
        e = cudaLaunchKernelEx(&cfg, block_norm_fwd_kernel<F32, false, 1024>, a);
    if (e != cudaSuccess) return fail(GDN_ERR_CUDA, "gdn_block_norm_fwd: launch failed: %s", cudaGetErrorString(e));
    return launch_status("gdn_block_norm_fwd");
}

// The ring of a wide backward row: as many stages as the SM's CTAs leave room for.
BwdRing bwd_ring(const BlockNormArgs& a, bool f32, bool row_gate) {
    BwdRing r;
    const int row = a.D * 2, hrow = a.D * (f32 ? 4 : 2);
    r.off_dx = row;
    r.off_h = r.off_dx + (a.gamma_pre ? row : 0);
    r.off_dh = r.off_h + (a.gamma_pre ? hrow : 0);
    r.off_gate = r.off_dh + (a.dh_out ? hrow : 0);
    r.bytes = r.off_gate + (row_gate ? row : 0);
    const int room = (220 * 1024) / bwd_resident(a.D) - (bwd_resident(a.D) > 1 ? 4096 : 0);
    r.stages = room / r.bytes < kMaxStages ? room / r.bytes : kMaxStages;
    return r;
}

template <bool F32>
int launch_bwd(const BlockNormArgs& a, const BwdPlan& p, void* dgate_rows, int dgate_f32, float* part_gamma,
               float* part_gate, cudaStream_t st) {
    const char* name = "gdn_block_norm_bwd";
    const int nt = block_threads(a.D);
    if (a.D <= kNarrow) {
        block_norm_bwd_narrow_kernel<F32>
            <<<p.ctas, nt, kNarrowRows * a.D * sizeof(float), st>>>(a, p, dgate_rows, dgate_f32, part_gamma, part_gate);
        return launch_status(name);
    }
    const BwdRing ring = bwd_ring(a, F32, dgate_rows != nullptr);
    const size_t smem = static_cast<size_t>(ring.stages) * ring.bytes;
    auto go = [&](auto kernel) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 221 * 1024);
        if (e != cudaSuccess) return fail(GDN_ERR_CUDA, "%s: cudaFuncSetAttribute: %s", name, cudaGetErrorString(e));
        kernel<<<p.ctas, nt, smem, st>>>(a, p, ring, dgate_rows, dgate_f32, part_gamma, part_gate);
        return launch_status(name);
    };
    if (nt <= 256) return go(block_norm_bwd_kernel<F32, 256>);
    if (nt <= 512) return go(block_norm_bwd_kernel<F32, 512>);
    return go(block_norm_bwd_kernel<F32, 1024>);
}

// Gate rows whose gradient is a sum (a gate row of its own for every row needs none).
int summed_gates(int R, int gate_rows) { return gate_rows > 0 && gate_rows < R ? gate_rows : 0; }

size_t bwd_bytes(int R, int D, int gate_rows) {
    const int sg = summed_gates(R, gate_rows);
    const BwdPlan p = bwd_plan(R, D, sg ? sg : 1);
    const size_t gamma = static_cast<size_t>(p.ctas) * 2 * D * sizeof(float);
    const size_t gate = sg ? static_cast<size_t>(p.groups) * p.parts * D * sizeof(float) : 0;
    return gamma + gate;
}

}  // namespace
}  // namespace gdn

extern "C" int gdn_block_norm_fwd(const void* y, const void* h, int h_dtype, const void* gamma_post, const void* gate,
                                  int gate_rows, const void* gamma_pre, float residual_scale, void* h_out, void* x,
                                  int R, int D, float eps, void* stream) {
    using namespace gdn;
    const char* name = "gdn_block_norm_fwd";
    int st = check_block_norm(name, y, h, h_dtype, gamma_post, gate, gate_rows, gamma_pre, R, D);
    if (st != GDN_OK) return st;
    if (!h_out || (gamma_pre && !x)) return fail(GDN_ERR_NULL, "%s: h_out, and x with gamma_pre, are required", name);
    if (!aligned16(h_out) || !aligned16(x)) return fail(GDN_ERR_ALIGN, "%s: pointers must be 16-byte aligned", name);
    if ((st = check_sm100()) != GDN_OK) return st;
    if (R == 0) return GDN_OK;
    BlockNormArgs a = {};
    a.y = static_cast<const uint16_t*>(y);
    a.h = h;
    a.gamma_post = static_cast<const uint16_t*>(gamma_post);
    a.gate = static_cast<const uint16_t*>(gate);
    a.gamma_pre = static_cast<const uint16_t*>(gamma_pre);
    a.h_out = h_out;
    a.x = static_cast<uint16_t*>(x);
    a.alpha = residual_scale;
    a.eps = eps;
    a.R = R;
    a.D = D;
    a.rows_per_gate = gate ? R / gate_rows : R;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return h_dtype == GDN_DTYPE_F32 ? launch_fwd<true>(a, s) : launch_fwd<false>(a, s);
}

extern "C" size_t gdn_block_norm_bwd_workspace_bytes(int R, int D, int gate_rows) {
    using namespace gdn;
    if (R <= 0 || D <= 0 || D % 8 != 0 || D > kMaxD || gate_rows < 0 || (gate_rows > 0 && R % gate_rows != 0)) return 0;
    return bwd_bytes(R, D, gate_rows);
}

extern "C" int gdn_block_norm_bwd(const void* y, const void* h_out, int h_dtype, const void* dh_out, const void* dx,
                                  const void* gamma_post, const void* gate, int gate_rows, const void* gamma_pre,
                                  float residual_scale, void* dy, void* dh, void* dgate, int dgate_dtype,
                                  float* dgamma_post, float* dgamma_pre, int R, int D, float eps, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    using namespace gdn;
    const char* name = "gdn_block_norm_bwd";
    int st = check_block_norm(name, y, h_out, h_dtype, gamma_post, gate, gate_rows, gamma_pre, R, D);
    if (st != GDN_OK) return st;
    if (!dy || !dh || (gamma_pre && (!dx || !dgamma_pre)) || (gamma_post && !dgamma_post) || (gate && !dgate))
        return fail(GDN_ERR_NULL, "%s: dy, dh, dx and dgamma_pre with gamma_pre, dgamma_post with gamma_post and dgate "
                                  "with a gate are required", name);
    if (gate && dgate_dtype != GDN_DTYPE_F32 && !(dgate_dtype == GDN_DTYPE_BF16 && gate_rows == R))
        return fail(GDN_ERR_DTYPE, "%s: dgate_dtype must be GDN_DTYPE_F32, or GDN_DTYPE_BF16 with gate_rows == R", name);
    for (const void* p : {static_cast<const void*>(dy), static_cast<const void*>(dh), static_cast<const void*>(dgate),
                          dh_out, dx, static_cast<const void*>(dgamma_post), static_cast<const void*>(dgamma_pre),
                          static_cast<const void*>(workspace)})
        if (!aligned16(p)) return fail(GDN_ERR_ALIGN, "%s: pointers must be 16-byte aligned", name);
    if (R > 0 && (!workspace || workspace_bytes < bwd_bytes(R, D, gate ? gate_rows : 0)))
        return fail(GDN_ERR_SHAPE, "%s: workspace of %zu bytes is smaller than %zu", name, workspace ? workspace_bytes : 0,
                    bwd_bytes(R, D, gate ? gate_rows : 0));
    if ((st = check_sm100()) != GDN_OK) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (R == 0) {                                        // no rows: the sums are zero
        cudaError_t e = cudaSuccess;
        if (gamma_post) e = cudaMemsetAsync(dgamma_post, 0, sizeof(float) * D, s);
        if (e == cudaSuccess && gamma_pre) e = cudaMemsetAsync(dgamma_pre, 0, sizeof(float) * D, s);
        if (e == cudaSuccess && gate) e = cudaMemsetAsync(dgate, 0, sizeof(float) * D * gate_rows, s);
        return e == cudaSuccess ? GDN_OK : fail(GDN_ERR_CUDA, "%s: cudaMemsetAsync: %s", name, cudaGetErrorString(e));
    }
    const int sg = gate ? summed_gates(R, gate_rows) : 0, groups = sg ? sg : 1;
    const BwdPlan p = bwd_plan(R, D, groups);
    BlockNormArgs a = {};
    a.y = static_cast<const uint16_t*>(y);
    a.h = h_out;
    a.gamma_post = static_cast<const uint16_t*>(gamma_post);
    a.gate = static_cast<const uint16_t*>(gate);
    a.gamma_pre = static_cast<const uint16_t*>(gamma_pre);
    a.h_out = dh;
    a.x = static_cast<uint16_t*>(dy);
    a.dh_out = dh_out;
    a.dx = static_cast<const uint16_t*>(dx);
    a.err = device_error_word();
    a.alpha = residual_scale;
    a.eps = eps;
    a.R = R;
    a.D = D;
    a.rows_per_gate = gate ? R / gate_rows : R;
    if (!gamma_pre) a.dx = nullptr;
    float* part_gamma = (gamma_post || gamma_pre) ? static_cast<float*>(workspace) : nullptr;
    float* part_gate = sg ? static_cast<float*>(workspace) + static_cast<size_t>(p.ctas) * 2 * D : nullptr;
    void* dgate_rows = gate && !sg ? dgate : nullptr;
    const int dgate_f32 = dgate_dtype == GDN_DTYPE_F32;
    st = h_dtype == GDN_DTYPE_F32 ? launch_bwd<true>(a, p, dgate_rows, dgate_f32, part_gamma, part_gate, s)
                                  : launch_bwd<false>(a, p, dgate_rows, dgate_f32, part_gamma, part_gate, s);
    if (st != GDN_OK) return st;
    if (!part_gamma && !part_gate) return GDN_OK;
    const SumJob j0 = {part_gamma, gamma_post ? dgamma_post : nullptr, 0, 2l * D, p.ctas};
    const SumJob j1 = {part_gamma ? part_gamma + D : nullptr, gamma_pre ? dgamma_pre : nullptr, 0, 2l * D, p.ctas};
    const SumJob j2 = {part_gate, part_gate ? static_cast<float*>(dgate) : nullptr, static_cast<long>(p.parts) * D, D, p.parts};
    cudaLaunchConfig_t cfg = {};                               // starts while the row kernel ends
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.stream = s;
    cfg.gridDim = dim3((D + 31) / 32, 2 + (part_gate ? (groups < kMaxGridY - 2 ? groups : kMaxGridY - 2) : 0));
    cfg.blockDim = dim3(32 * kSumWarps);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, column_sum_kernel, j0, j1, j2, groups, D);
    if (e != cudaSuccess) return fail(GDN_ERR_CUDA, "%s: launch failed: %s", name, cudaGetErrorString(e));
    return launch_status("gdn_block_norm_bwd (column sums)");
}
