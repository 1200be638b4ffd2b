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
// belong to one warp (shuffles only), wider ones to a CTA.
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
__device__ __forceinline__ void load8_bf16(const uint16_t* p, float (&f)[8]) {
    unpack8(__ldcg(reinterpret_cast<const uint4*>(p)), f);
}
__device__ __forceinline__ void store8_bf16(uint16_t* p, const float (&f)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                              pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}
template <bool F32>
__device__ __forceinline__ void load8(const void* base, long at, float (&f)[8]) {
    if constexpr (F32) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
        const float4 a = __ldcg(p), b = __ldcg(p + 1);
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
        f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
        load8_bf16(static_cast<const uint16_t*>(base) + at, f);
    }
}
template <bool F32>
__device__ __forceinline__ void store8(void* base, long at, const float (&f)[8]) {
    if constexpr (F32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + at);
        p[0] = make_float4(f[0], f[1], f[2], f[3]);
        p[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
        store8_bf16(static_cast<uint16_t*>(base) + at, f);
    }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum of N values over the row's threads: one warp, or the whole CTA through `red`
// ([2][N][32] floats, used in turn so that one barrier per sum is enough).
template <int N, bool WARP>
__device__ __forceinline__ void row_sum(float (&v)[N], float* red, int& turn) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
    if constexpr (!WARP) {
        float* mine = red + turn * (N * 32);
        turn ^= 1;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) mine[i * 32 + warp] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < nw ? mine[i * 32 + lane] : 0.f);
    }
}

template <bool F32, bool WARP, int NT>
__global__ void __launch_bounds__(NT) block_norm_fwd_kernel(const BlockNormArgs a) {
    __shared__ float red[2][32];
    pdl_launch_dependents();
    pdl_wait_prior();                          // y and h come from earlier kernels
    const int piece = WARP ? (threadIdx.x & 31) : threadIdx.x;
    const bool on = piece * 8 < a.D;
    const long row0 = WARP ? static_cast<long>(blockIdx.x) * kNarrowRows + (threadIdx.x >> 5) : blockIdx.x;
    const long step = WARP ? static_cast<long>(gridDim.x) * kNarrowRows : gridDim.x;
    const float inv_d = 1.f / static_cast<float>(a.D);
    int turn = 0;
    for (long r = row0; r < a.R; r += step) {
        const long at = r * a.D + piece * 8;
        float u[8] = {}, h[8] = {}, w[8];
        if (on) {
            load8_bf16(a.y + at, u);
            load8<F32>(a.h, at, h);
        }
        if (a.gamma_post) {
            float ss[1] = {0.f};
#pragma unroll
            for (int i = 0; i < 8; ++i) ss[0] += u[i] * u[i];
            row_sum<1, WARP>(ss, &red[0][0], turn);
            const float r1 = rsqrtf(ss[0] * inv_d + a.eps);
            if (on) {
                unpack8(__ldg(reinterpret_cast<const uint4*>(a.gamma_post + piece * 8)), w);
#pragma unroll
                for (int i = 0; i < 8; ++i) u[i] *= r1 * w[i];
            }
        }
        if (a.gate && on) {
            load8_bf16(a.gate + (r / a.rows_per_gate) * a.D + piece * 8, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] *= w[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = fmaf(a.alpha, h[i], u[i]);
        if (on) store8<F32>(a.h_out, at, h);
        if (a.gamma_pre) {
            float ss[1] = {0.f};
#pragma unroll
            for (int i = 0; i < 8; ++i) ss[0] += h[i] * h[i];
            row_sum<1, WARP>(ss, &red[0][0], turn);
            const float r2 = rsqrtf(ss[0] * inv_d + a.eps);
            if (on) {
                unpack8(__ldg(reinterpret_cast<const uint4*>(a.gamma_pre + piece * 8)), w);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[i] *= r2 * w[i];
                store8_bf16(a.x + at, h);
            }
        }
    }
}

// The rows a backward work item covers: one of `per_gate` parts of one gate row's rows,
// so the column sums of an item belong to one gate row.
struct BwdPlan {
    int groups;                       // gate rows that are summed over rows (1 when none are)
    int parts;                        // parts per group
    int ctas;
};

// dgamma partials: [ctas][2][D]; dgate partials: [groups * parts][D] (after them).
template <bool F32, bool WARP, int NT>
__global__ void __launch_bounds__(NT)
block_norm_bwd_kernel(const BlockNormArgs a, const BwdPlan plan, void* dgate_rows, int dgate_f32, float* part_gamma,
                      float* part_gate) {
    __shared__ float red[2][2][32];
    __shared__ float red1[2][32];
    const int piece = WARP ? (threadIdx.x & 31) : threadIdx.x;
    const int sub = WARP ? (threadIdx.x >> 5) : 0, nsub = WARP ? kNarrowRows : 1;
    const bool on = piece * 8 < a.D;
    const float inv_d = 1.f / static_cast<float>(a.D);
    const int items = plan.groups * plan.parts;
    const long group_rows = a.R / plan.groups;
    const int col = piece * 8;
    int turn = 0, turn1 = 0;
    float gp[8], gq[8], sum_post[8] = {}, sum_pre[8] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) gp[i] = gq[i] = 1.f;
    if (on && a.gamma_post) unpack8(__ldg(reinterpret_cast<const uint4*>(a.gamma_post + col)), gp);
    if (on && a.gamma_pre) unpack8(__ldg(reinterpret_cast<const uint4*>(a.gamma_pre + col)), gq);
    extern __shared__ float cols[];            // WARP: [rows of the CTA][D] for the column sums
    // sum over the CTA's warps of the lanes' 8 columns, in warp order, into dst (WARP only)
    auto write_cols = [&](const float (&v)[8], float* dst) {
        if constexpr (WARP) {
            __syncthreads();
            if (on)
#pragma unroll
                for (int i = 0; i < 8; ++i) cols[sub * a.D + col + i] = v[i];
            __syncthreads();
            for (int c = threadIdx.x; c < a.D; c += blockDim.x) {
                float s = 0.f;
                for (int w = 0; w < kNarrowRows; ++w) s += cols[w * a.D + c];
                dst[c] = s;
            }
        } else if (on) {
            float4* p = reinterpret_cast<float4*>(dst + col);
            p[0] = make_float4(v[0], v[1], v[2], v[3]);
            p[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
    };
    for (int it = blockIdx.x; it < items; it += gridDim.x) {
        const int g = it / plan.parts, part = it % plan.parts;
        const long r0 = g * group_rows + group_rows * part / plan.parts;
        const long r1_ = g * group_rows + group_rows * (part + 1) / plan.parts;
        float sum_gate[8] = {};
        // every warp of the CTA runs the same number of turns (WARP has no barrier in the loop)
        for (long r = r0 + sub; r < r1_; r += nsub) {
            const long at = r * a.D + col;
            float y[8] = {}, h[8] = {}, dx[8] = {}, dt[8] = {}, gt[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) gt[i] = 1.f;
            if (on) {
                load8_bf16(a.y + at, y);
                load8<F32>(a.h, at, h);
                if (a.gamma_pre) load8_bf16(a.dx + at, dx);
                if (a.dh_out) load8<F32>(a.dh_out, at, dt);
                if (a.gate) load8_bf16(a.gate + (r / a.rows_per_gate) * a.D + col, gt);
            }
            float s[2] = {0.f, 0.f}, s2[1] = {0.f};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s[0] += y[i] * y[i];
                s[1] += h[i] * h[i];
            }
            row_sum<2, WARP>(s, &red[0][0][0], turn);
            if (a.gamma_pre) {
                const float r2 = rsqrtf(s[1] * inv_d + a.eps);
                float m[1] = {0.f};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    h[i] *= r2;                                 // n2
                    sum_pre[i] += dx[i] * h[i];
                    dx[i] *= gq[i];                             // g2
                    m[0] += dx[i] * h[i];
                }
                row_sum<1, WARP>(m, &red1[0][0], turn1);
                m[0] *= inv_d;
#pragma unroll
                for (int i = 0; i < 8; ++i) dt[i] += r2 * (dx[i] - h[i] * m[0]);
            }
            const float r1 = a.gamma_post ? rsqrtf(s[0] * inv_d + a.eps) : 1.f;
            float dg[8], out[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y[i] *= r1;                                     // n1
                dg[i] = dt[i] * y[i] * gp[i];
                out[i] = a.alpha * dt[i];
                dt[i] *= gt[i];                                 // du
                sum_post[i] += dt[i] * y[i];
                sum_gate[i] += dg[i];
                dt[i] *= gp[i];                                 // g1
                s2[0] += dt[i] * y[i];
            }
            if (on) {
                store8<F32>(a.h_out, at, out);
                if (dgate_rows) {
                    if (dgate_f32)
                        store8<true>(dgate_rows, at, dg);
                    else
                        store8<false>(dgate_rows, at, dg);
                }
            }
            if (a.gamma_post) {
                row_sum<1, WARP>(s2, &red1[0][0], turn1);
                s2[0] *= inv_d;
#pragma unroll
                for (int i = 0; i < 8; ++i) dt[i] = r1 * (dt[i] - y[i] * s2[0]);
            }
            if (on) store8_bf16(a.x + at, dt);
        }
        if (part_gate) write_cols(sum_gate, part_gate + static_cast<long>(it) * a.D);
    }
    if (part_gamma) {
        write_cols(sum_post, part_gamma + (static_cast<long>(blockIdx.x) * 2) * a.D);
        write_cols(sum_pre, part_gamma + (static_cast<long>(blockIdx.x) * 2 + 1) * a.D);
    }
}

// out[o][c] = sum over n of in[(o * n_stride_o + n * n_stride)][c], in the order of n:
// 32 columns x 8 partial sums a CTA, then their sum in order.
struct SumJob {
    const float* in;
    float* out;
    long o_stride, n_stride;          // elements
    int n;
};
__global__ void __launch_bounds__(256) column_sum_kernel(const SumJob j0, const SumJob j1, const SumJob j2, int D) {
    __shared__ float part[8][32];
    // blockIdx.y 0: dgamma_post, 1: dgamma_pre, 2 + g: gate row g
    const SumJob& j = blockIdx.y == 0 ? j0 : blockIdx.y == 1 ? j1 : j2;
    if (!j.out) return;
    const long o = blockIdx.y < 2 ? 0 : blockIdx.y - 2;
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
    float s = 0.f;
    if (c < D) {
        const float* p = j.in + o * j.o_stride + c;
        for (int n = k; n < j.n; n += 8) s += __ldcg(p + n * j.n_stride);
    }
    part[k][threadIdx.x & 31] = s;
    __syncthreads();
    if (k == 0 && c < D) {
        for (int i = 1; i < 8; ++i) s += part[i][threadIdx.x & 31];
        j.out[o * D + c] = s;
    }
}

int block_threads(int D) { return D <= kNarrow ? 32 * kNarrowRows : (D / 8 + 31) / 32 * 32; }

// `groups`: gate rows whose gradient is a sum over rows (1 without such a sum).
BwdPlan bwd_plan(int R, int D, int groups) {
    BwdPlan p;
    p.groups = groups;
    const int per_cta = D <= kNarrow ? kNarrowRows : 1;
    const int resident = 2048 / block_threads(D) > 4 ? 4 : 2048 / block_threads(D);
    const int want = 148 * (resident < 1 ? 1 : resident);
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
    cfg.gridDim = dim3((a.R + rows - 1) / rows);
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

template <bool F32>
int launch_bwd(const BlockNormArgs& a, const BwdPlan& p, void* dgate_rows, int dgate_f32, float* part_gamma,
               float* part_gate, cudaStream_t st) {
    const int nt = block_threads(a.D);
    if (a.D <= kNarrow)
        block_norm_bwd_kernel<F32, true, 256>
            <<<p.ctas, nt, kNarrowRows * a.D * sizeof(float), st>>>(a, p, dgate_rows, dgate_f32, part_gamma, part_gate);
    else if (nt <= 256)
        block_norm_bwd_kernel<F32, false, 256><<<p.ctas, nt, 0, st>>>(a, p, dgate_rows, dgate_f32, part_gamma, part_gate);
    else if (nt <= 512)
        block_norm_bwd_kernel<F32, false, 512><<<p.ctas, nt, 0, st>>>(a, p, dgate_rows, dgate_f32, part_gamma, part_gate);
    else
        block_norm_bwd_kernel<F32, false, 1024><<<p.ctas, nt, 0, st>>>(a, p, dgate_rows, dgate_f32, part_gamma, part_gate);
    return launch_status("gdn_block_norm_bwd");
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
    if (groups > 65533) return fail(GDN_ERR_SHAPE, "%s: at most 65533 gate rows that are shared (got %d)", name, groups);
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
    a.alpha = residual_scale;
    a.eps = eps;
    a.R = R;
    a.D = D;
    a.rows_per_gate = gate ? R / gate_rows : R;
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
    const dim3 grid((D + 31) / 32, 2 + (part_gate ? groups : 0));
    column_sum_kernel<<<grid, 256, 0, s>>>(j0, j1, j2, D);
    return launch_status("gdn_block_norm_bwd (column sums)");
}
