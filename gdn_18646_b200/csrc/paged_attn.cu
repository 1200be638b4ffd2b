// paged_attn.cu -- softmax attention of new tokens over a paged key/value cache.
//
// Token i of sequence b stands at position p = kv_len - q_len + i and sees the positions
// lo .. hi of its mask; one pass over them with the running maximum m and sum l of the
// softmax (fp32):
//   s_j = scale q.k_j,  m' = max(m, s_j),  l' = l e^(m-m') + e^(s_j-m'),
//   o' = o e^(m-m') + e^(s_j-m') v_j;   out = o / l, lse = m + log l
// A row that sees nothing keeps l = 0: out 0, lse -inf.
#include "common.cuh"
#include "paged.cuh"

namespace gdn {
namespace {

constexpr int kWarps = 4;

struct AttnArgs {
    const uint16_t* q;
    long q_ld;
    uint16_t* out;
    float* lse;
    PagedView cache;
    const int* cu;
    const int* kv_lens;
    int B, T, Hq, group;
    int max_q, max_kv;
    int causal, window;
    float scale;
    unsigned int* err;
};

// One warp per (token, query head); a lane owns D/32 consecutive values of a row.
template <int D>
__global__ void __launch_bounds__(32 * kWarps) paged_attn_rows_kernel(const AttnArgs a) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31;
    const long job = static_cast<long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    if (job >= static_cast<long>(a.T) * a.Hq) return;
    const int t = static_cast<int>(job / a.Hq), h = static_cast<int>(job % a.Hq), kh = h / a.group;
    const int b = sequence_of(a.cu, a.B, t);
    const int c0 = a.cu[b], c1 = a.cu[b + 1];
    int len = a.kv_lens[b];
    if (t < c0 || t >= c1 || c0 < 0 || c1 > a.T || c1 - c0 > a.max_q || len > a.max_kv || len < 0) {
        if (lane == 0) atomicOr(a.err, DERR_PAGED);
        len = min(max(len, 0), a.max_kv);
    }
    const int pos = len - c1 + t;
    int hi = a.causal ? min(pos + 1, len) : len, lo = 0;
    if (a.window > 0) lo = max(0, pos + 1 - a.window);
    const uint16_t* qp = a.q + t * a.q_ld + h * D + lane * V;
    float q[V], o[V] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) q[i] = bf16_bits_to_f32(qp[i]) * a.scale;
    for (int j = lo; j < hi; ++j) {
        const int page = a.cache.table[b * a.cache.table_ld + (j >> a.cache.page_shift)];
        if (page < 0 || page >= a.cache.num_pages) {
            if (lane == 0) atomicOr(a.err, DERR_PAGED);
        }
        const bool have = page >= 0 && page < a.cache.num_pages;
        const long at = (have ? page : 0) * a.cache.page_stride +
                        (j & ((1 << a.cache.page_shift) - 1)) * a.cache.token_stride + kh * a.cache.head_stride + lane * V;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) s += q[i] * (have ? bf16_bits_to_f32(a.cache.k[at + i]) : 0.f);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        const float mn = fmaxf(m, s);
        if (mn == -INFINITY) continue;
        const float c = __expf(m - mn), p = __expf(s - mn);
        m = mn;
        l = l * c + p;
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = o[i] * c + p * (have ? bf16_bits_to_f32(a.cache.v[at + i]) : 0.f);
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    uint16_t* op = a.out + (static_cast<long>(t) * a.Hq + h) * D + lane * V;
#pragma unroll
    for (int i = 0; i < V; ++i) op[i] = f32_to_bf16_bits(l > 0.f ? o[i] * inv : 0.f);
    if (a.lse && lane == 0) a.lse[static_cast<long>(t) * a.Hq + h] = l > 0.f ? m + logf(l) : -INFINITY;
}

}  // namespace
}  // namespace gdn

extern "C" size_t gdn_paged_attn_workspace_bytes(int B, int Ttot, int Hq, int n_kv, int head_dim, int max_q, int max_kv,
                                                 int window) {
    (void)B, (void)Ttot, (void)Hq, (void)n_kv, (void)head_dim, (void)max_q, (void)max_kv, (void)window;
    return 0;
}

extern "C" int gdn_paged_attn_fwd(const void* q, long q_ld, const gdn_paged_cache* cache, const int* cu_seqlens,
                                  const int* kv_lens, void* out, float* lse, int B, int Ttot, int Hq, int max_q,
                                  int max_kv, int causal, int window, float scale, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    using namespace gdn;
    const char* name = "gdn_paged_attn_fwd";
    (void)workspace, (void)workspace_bytes;
    AttnArgs a = {};
    int st = check_cache(name, cache, &a.cache);
    if (st != GDN_OK) return st;
    if (!q || !cu_seqlens || !kv_lens || !out)
        return fail(GDN_ERR_NULL, "%s: q, cu_seqlens, kv_lens and out are required", name);
    const int D = cache->head_dim;
    if (D != 64 && D != 128) return fail(GDN_ERR_UNSUPPORTED, "%s: head dim %d (64 or 128)", name, D);
    if (B < 1 || Ttot < 0 || Hq < 1 || max_q < 0 || max_kv < 0)
        return fail(GDN_ERR_SHAPE, "%s: B=%d Ttot=%d Hq=%d max_q=%d max_kv=%d", name, B, Ttot, Hq, max_q, max_kv);
    if (Hq % cache->n_kv != 0 || Hq / cache->n_kv > 64)
        return fail(GDN_ERR_SHAPE, "%s: Hq=%d must be a multiple, at most 64 times, of n_kv=%d", name, Hq, cache->n_kv);
    if (max_kv > cache->max_pages * cache->page_size)
        return fail(GDN_ERR_SHAPE, "%s: max_kv=%d exceeds the %d positions of a block_table row", name, max_kv,
                    cache->max_pages * cache->page_size);
    if (Ttot > 1 && q_ld < static_cast<long>(Hq) * D) return fail(GDN_ERR_SHAPE, "%s: q rows of %ld elements overlap", name, q_ld);
    if (window < 0 || (window > 0 && !causal)) return fail(GDN_ERR_ARG, "%s: a window needs causal, and must not be negative", name);
    if (!aligned16(q) || !aligned16(out) || q_ld % 8 != 0)
        return fail(GDN_ERR_ALIGN, "%s: q, its rows and out must be 16-byte aligned", name);
    if ((st = check_sm100()) != GDN_OK) return st;
    if (Ttot == 0) return GDN_OK;
    a.q = static_cast<const uint16_t*>(q);
    a.q_ld = q_ld;
    a.out = static_cast<uint16_t*>(out);
    a.lse = lse;
    a.cu = cu_seqlens;
    a.kv_lens = kv_lens;
    a.B = B;
    a.T = Ttot;
    a.Hq = Hq;
    a.group = Hq / cache->n_kv;
    a.max_q = max_q;
    a.max_kv = max_kv;
    a.causal = causal != 0;
    a.window = window;
    a.scale = scale == 0.f ? 1.f / sqrtf(static_cast<float>(D)) : scale;
    a.err = device_error_word();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const long jobs = static_cast<long>(Ttot) * Hq;
    const unsigned grid = static_cast<unsigned>((jobs + kWarps - 1) / kWarps);
    if (D == 64)
        paged_attn_rows_kernel<64><<<grid, 32 * kWarps, 0, s>>>(a);
    else
        paged_attn_rows_kernel<128><<<grid, 32 * kWarps, 0, s>>>(a);
    return launch_status(name);
}
