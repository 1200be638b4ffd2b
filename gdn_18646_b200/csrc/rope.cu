// rope.cu -- rotary positions with several axes, and the same with the append of the
// new keys and values to a paged cache.
//
//   angle(t, i) = positions[axis(i)][t] * inv_freq[i]        i < rot / 2
//   (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin)           (inverse: -sin)
//
// Bound by HBM: every head row is read once and written once.  A warp takes a token;
// its lanes split into groups of D/16, each lane holding the 8 pairs (16 values, two
// 16-byte pieces) of one unit of a head, so the 8 sines and cosines that a lane needs
// are the same for every head it turns and are computed once.  269 MB of q and k turned:
// 42.0 us, 6.4 TB/s; 112 MB of q, k, v appended (11 K tokens): 22.0 us, 5.1 TB/s, held back by
// the chain token -> sequence -> page -> address before a token's first store.
//
// The angle is reduced in fp32 with the product's rounding error carried along
// (pos * f = hi + lo exactly by an fma) and 2 pi in two parts, after Cody and Waite, so the
// angle is off by at most 8.1e-7 rad for positions up to 2^24 (the same steps on the CPU
// against 64 bits, 10^7 pairs), where the rounded product alone would lose 0.03 at 10^6 and
// 0.5 at 2^24; by 1.3e-5 at 2^30 and 2.6e-5 at 2^31.  sin and cos of the reduced angle then are
// the fast intrinsics (absolute error 2^-21, against the 2^-9 of a bf16 result).
#include "common.cuh"
#include "paged.cuh"

namespace gdn {
namespace {

constexpr int kMaxAxes = 4;
constexpr int kWarps = 4;             // warps (tokens, or parts of a token's heads) per CTA

struct RopeArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;                // append only
    uint16_t* q_out;
    uint16_t* k_out;                  // rope only
    long q_ld, k_ld, v_ld;
    const int* positions;
    long positions_ld;
    const float* inv_freq;
    int bound[kMaxAxes];              // first pair past axis a
    int axes, half;                   // half = rot / 2
    int T, Hq, Hk;
    int splits;                       // warps that share a token's heads
    float sign;
    // append
    PagedView cache;
    const int* cu;
    const int* kv_lens;
    int B;
    unsigned int* err;
};

__device__ __forceinline__ void sincos_of(int pos, float f, float sign, float& s, float& c) {
    constexpr float kInv2Pi = 0.15915494309189535f;
    constexpr float k2PiHi = 6.2831854820251465f;          // 2 pi rounded to fp32
    constexpr float k2PiLo = -1.7484556000744883e-07f;     // 2 pi - k2PiHi
    // a position past 2^24 is split so that both parts are exact
    const float p1 = static_cast<float>(pos & ~0xfff), p0 = static_cast<float>(pos & 0xfff);
    float hi = p1 * f, lo = fmaf(p1, f, -hi);
    float n = rintf(hi * kInv2Pi);
    float r = fmaf(-n, k2PiHi, hi);
    r = fmaf(-n, k2PiLo, r) + lo;
    hi = p0 * f;
    lo = fmaf(p0, f, -hi);
    n = rintf(hi * kInv2Pi);
    float r0 = fmaf(-n, k2PiHi, hi);
    r0 = fmaf(-n, k2PiLo, r0) + lo;
    r += r0;                                               // |r| <= 2 pi
    n = rintf(r * kInv2Pi);
    r = fmaf(-n, k2PiHi, r);
    __sincosf(r, &s, &c);
    s *= sign;
}

__device__ __forceinline__ void unpack8(const uint4& w, float (&f)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(u[i] << 16);
        f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
}

template <int D, bool INTERLEAVED, bool APPEND>
__global__ void __launch_bounds__(32 * kWarps) rope_kernel(const RopeArgs a) {
    constexpr int UNITS = D / 16;              // lanes per head
    constexpr int HPW = 32 / UNITS;            // heads a warp turns at once
    // such groups of heads whose loads are in flight together (us at 11 K tokens of 20 heads, with 3
    // and 5: append 23.1, 22.0; at 16 K tokens of 32 heads: plain 44.0, 45.9)
    constexpr int BATCH = APPEND ? 5 : 3;
    const int lane = threadIdx.x & 31, unit = lane % UNITS, sub = lane / UNITS;
    const uint32_t job = blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int t = static_cast<int>(job / a.splits), split = static_cast<int>(job - t * a.splits);
    if (t >= a.T) return;
    const bool turn = unit * 8 < a.half;
    // the two 16-byte pieces of this lane's unit: of a rotated unit (pieces p0, p1) and of a copied one
    const int p0 = (turn && !INTERLEAVED) ? unit * 8 : unit * 16;
    const int p1 = (turn && !INTERLEAVED) ? a.half + unit * 8 : unit * 16 + 8;
    const int heads = a.Hq + a.Hk * (APPEND ? 2 : 1), step = a.splits * HPW;
    const int h0 = split * HPW + sub;
    uint4 w[BATCH][2];
    auto load = [&](int h, uint4 (&x)[2]) {
        const uint16_t* src;
        if (h < a.Hq)
            src = a.q + t * a.q_ld + h * D;
        else if (h < a.Hq + a.Hk)
            src = a.k + t * a.k_ld + (h - a.Hq) * D;
        else
            src = a.v + t * a.v_ld + (h - a.Hq - a.Hk) * D;
        x[0] = __ldcg(reinterpret_cast<const uint4*>(src + p0));
        x[1] = __ldcg(reinterpret_cast<const uint4*>(src + p1));
    };
    // the first heads' loads are in flight while the token's place and its angles are found
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
        if (h0 + i * step < heads) load(h0 + i * step, w[i]);

    int pos[kMaxAxes] = {};
    if (turn) {
#pragma unroll
        for (int x = 0; x < kMaxAxes; ++x)
            if (x < a.axes) pos[x] = a.positions[x * a.positions_ld + t];
    }
    // where this token's key and value go
    long slot = -1;
    if constexpr (APPEND) {
        const int b = sequence_of(a.cu, a.B, t);
        const int c0 = a.cu[b], c1 = a.cu[b + 1], len = a.kv_lens[b];
        const int at = len - c1 + t;
        const int pg = at >> a.cache.page_shift;
        bool ok = t >= c0 && t < c1 && c0 >= 0 && len >= 0 && at >= 0 && at < len && pg < a.cache.max_pages;
        if (ok) {
            const int page = a.cache.table[b * a.cache.table_ld + pg];
            ok = page >= 0 && page < a.cache.num_pages;
            slot = page * a.cache.page_stride + (at & ((1 << a.cache.page_shift) - 1)) * a.cache.token_stride;
        }
        if (!ok) {
            slot = -1;
            if (lane == 0 && split == 0) atomicOr(a.err, DERR_PAGED);
        }
    }
    float sn[8], cs[8];
    if (turn) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int pair = unit * 8 + i;
            int p = pos[0];
#pragma unroll
            for (int x = 1; x < kMaxAxes; ++x)
                if (x < a.axes && pair >= a.bound[x - 1]) p = pos[x];
            sincos_of(p, __ldg(a.inv_freq + pair), a.sign, sn[i], cs[i]);
        }
    }
    auto finish = [&](int h, uint4 (&x)[2]) {
        uint16_t* dst;
        if (h < a.Hq) {
            dst = a.q_out + (static_cast<long>(t) * a.Hq + h) * D;
        } else if constexpr (!APPEND) {
            dst = a.k_out + (static_cast<long>(t) * a.Hk + (h - a.Hq)) * D;
        } else {
            if (slot < 0) return;
            dst = h < a.Hq + a.Hk ? a.cache.k + slot + (h - a.Hq) * a.cache.head_stride
                                  : a.cache.v + slot + (h - a.Hq - a.Hk) * a.cache.head_stride;
        }
        if (turn && h < a.Hq + a.Hk) {
            float x0[8], x1[8];
            unpack8(x[0], x0);
            unpack8(x[1], x1);
            if constexpr (INTERLEAVED) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = x0[2 * i], f = x0[2 * i + 1], g = x1[2 * i], k = x1[2 * i + 1];
                    x0[2 * i] = e * cs[i] - f * sn[i];
                    x0[2 * i + 1] = f * cs[i] + e * sn[i];
                    x1[2 * i] = g * cs[i + 4] - k * sn[i + 4];
                    x1[2 * i + 1] = k * cs[i + 4] + g * sn[i + 4];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float e = x0[i], f = x1[i];
                    x0[i] = e * cs[i] - f * sn[i];
                    x1[i] = f * cs[i] + e * sn[i];
                }
            }
            x[0] = pack8(x0);
            x[1] = pack8(x1);
        }
        *reinterpret_cast<uint4*>(dst + p0) = x[0];
        *reinterpret_cast<uint4*>(dst + p1) = x[1];
    };
    for (int h = h0; h < heads; h += BATCH * step) {
        if (h != h0)
#pragma unroll
            for (int i = 0; i < BATCH; ++i)
                if (h + i * step < heads) load(h + i * step, w[i]);
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
            if (h + i * step < heads) finish(h + i * step, w[i]);
    }
}

int check_rope(const char* name, const gdn_rope_spec* s, int D, RopeArgs* a) {
    if (!s || !s->positions || !s->inv_freq || !s->sections)
        return fail(GDN_ERR_NULL, "%s: the spec's positions, inv_freq and sections are required", name);
    if (D != 64 && D != 128 && D != 256) return fail(GDN_ERR_UNSUPPORTED, "%s: head dim %d (64, 128 or 256)", name, D);
    if (s->rot <= 0 || s->rot > D || s->rot % 16 != 0)
        return fail(GDN_ERR_SHAPE, "%s: rot must be a multiple of 16 in (0, %d] (got %d)", name, D, s->rot);
    if (s->axes < 1 || s->axes > kMaxAxes) return fail(GDN_ERR_SHAPE, "%s: 1 to %d axes (got %d)", name, kMaxAxes, s->axes);
    if (s->style != GDN_ROPE_HALF && s->style != GDN_ROPE_INTERLEAVED)
        return fail(GDN_ERR_ARG, "%s: style must be GDN_ROPE_HALF or GDN_ROPE_INTERLEAVED", name);
    long sum = 0;
    for (int i = 0; i < s->axes; ++i) {
        if (s->sections[i] < 0) return fail(GDN_ERR_SHAPE, "%s: sections must not be negative", name);
        sum += s->sections[i];
        a->bound[i] = static_cast<int>(sum);
    }
    if (sum != s->rot / 2) return fail(GDN_ERR_SHAPE, "%s: sections must sum to rot / 2 = %d (got %ld)", name, s->rot / 2, sum);
    a->positions = s->positions;
    a->positions_ld = s->positions_ld;
    a->inv_freq = s->inv_freq;
    a->axes = s->axes;
    a->half = s->rot / 2;
    return GDN_OK;
}

int check_rows(const char* name, const char* what, const void* p, long ld, int H, int D, int T) {
    if (!p) return fail(GDN_ERR_NULL, "%s: %s is required", name, what);
    if (!aligned16(p) || ld % 8 != 0) return fail(GDN_ERR_ALIGN, "%s: %s must be 16-byte aligned, its rows too", name, what);
    if (T > 1 && ld < static_cast<long>(H) * D) return fail(GDN_ERR_SHAPE, "%s: %s rows of %ld elements overlap", name, what, ld);
    return GDN_OK;
}

// Warps per token: few tokens are spread over warps by groups of heads, down to one group
// each, as latency counts.  With tokens enough for the GPU a warp of the append takes a
// token whole (finding its page costs more than its heads: 11 K tokens 23.1 us with one warp a
// token, 23.7 with two, 33.6 with three), of the plain rotation about half of one (16 K
// tokens 44.0 us with one warp, 42.0 with two, 42.5 with three).
int splits_for(int T, int heads, int D, bool append) {
    const int groups = (heads + 512 / D - 1) / (512 / D), warps = 148 * (append ? 16 : 128);
    const int want = T >= warps ? 1 : (warps + T - 1) / T;
    return want < groups ? want : groups;
}

template <bool APPEND>
int launch(const char* name, RopeArgs& a, int style, int D, cudaStream_t st) {
    a.splits = splits_for(a.T, a.Hq + a.Hk * (APPEND ? 2 : 1), D, APPEND);
    const long jobs = static_cast<long>(a.T) * a.splits;
    const dim3 grid(static_cast<unsigned>((jobs + kWarps - 1) / kWarps));
#define GDN_ROPE(DD)                                                                              \
    if (D == DD) {                                                                                \
        if (style == GDN_ROPE_INTERLEAVED)                                                        \
            rope_kernel<DD, true, APPEND><<<grid, 32 * kWarps, 0, st>>>(a);                       \
        else                                                                                      \
            rope_kernel<DD, false, APPEND><<<grid, 32 * kWarps, 0, st>>>(a);                      \
    }
    GDN_ROPE(64)
    GDN_ROPE(128)
    GDN_ROPE(256)
#undef GDN_ROPE
    return launch_status(name);
}

}  // namespace
}  // namespace gdn

extern "C" int gdn_rope_fwd(const void* q, long q_ld, const void* k, long k_ld, void* q_out, void* k_out,
                            const gdn_rope_spec* spec, int inverse, int T, int Hq, int Hk, int D, void* stream) {
    using namespace gdn;
    const char* name = "gdn_rope_fwd";
    RopeArgs a = {};
    int st = check_rope(name, spec, D, &a);
    if (st != GDN_OK) return st;
    if (T < 0 || Hq < 1 || Hk < 0) return fail(GDN_ERR_SHAPE, "%s: T=%d Hq=%d Hk=%d", name, T, Hq, Hk);
    if ((st = check_rows(name, "q", q, q_ld, Hq, D, T)) != GDN_OK) return st;
    if (Hk > 0 && (st = check_rows(name, "k", k, k_ld, Hk, D, T)) != GDN_OK) return st;
    if (!q_out || (Hk > 0 && !k_out)) return fail(GDN_ERR_NULL, "%s: q_out and k_out are required", name);
    if (!aligned16(q_out) || !aligned16(k_out)) return fail(GDN_ERR_ALIGN, "%s: outputs must be 16-byte aligned", name);
    if (T > 0 && a.axes > 1 && spec->positions_ld < T) return fail(GDN_ERR_SHAPE, "%s: positions_ld=%ld below T=%d", name, spec->positions_ld, T);
    if ((st = check_sm100()) != GDN_OK) return st;
    if (T == 0) return GDN_OK;
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.q_out = static_cast<uint16_t*>(q_out);
    a.k_out = static_cast<uint16_t*>(k_out);
    a.q_ld = q_ld;
    a.k_ld = k_ld;
    a.T = T;
    a.Hq = Hq;
    a.Hk = Hk;
    a.sign = inverse ? -1.f : 1.f;
    return launch<false>(name, a, spec->style, D, static_cast<cudaStream_t>(stream));
}

extern "C" int gdn_rope_append(const void* q, long q_ld, const void* k, long k_ld, const void* v, long v_ld, void* q_out,
                               const gdn_rope_spec* spec, const gdn_paged_cache* cache, const int* cu_seqlens,
                               const int* kv_lens, int B, int T, int Hq, void* stream) {
    using namespace gdn;
    const char* name = "gdn_rope_append";
    RopeArgs a = {};
    int st = check_cache(name, cache, &a.cache);
    if (st != GDN_OK) return st;
    const int D = cache->head_dim, Hk = cache->n_kv;
    if ((st = check_rope(name, spec, D, &a)) != GDN_OK) return st;
    if (T < 0 || Hq < 1 || B < 1) return fail(GDN_ERR_SHAPE, "%s: T=%d Hq=%d B=%d", name, T, Hq, B);
    if ((st = check_rows(name, "q", q, q_ld, Hq, D, T)) != GDN_OK) return st;
    if ((st = check_rows(name, "k", k, k_ld, Hk, D, T)) != GDN_OK) return st;
    if ((st = check_rows(name, "v", v, v_ld, Hk, D, T)) != GDN_OK) return st;
    if (!q_out || !cu_seqlens || !kv_lens) return fail(GDN_ERR_NULL, "%s: q_out, cu_seqlens and kv_lens are required", name);
    if (!aligned16(q_out)) return fail(GDN_ERR_ALIGN, "%s: q_out must be 16-byte aligned", name);
    if (T > 0 && a.axes > 1 && spec->positions_ld < T) return fail(GDN_ERR_SHAPE, "%s: positions_ld=%ld below T=%d", name, spec->positions_ld, T);
    if ((st = check_sm100()) != GDN_OK) return st;
    if (T == 0) return GDN_OK;
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.q_out = static_cast<uint16_t*>(q_out);
    a.q_ld = q_ld;
    a.k_ld = k_ld;
    a.v_ld = v_ld;
    a.T = T;
    a.Hq = Hq;
    a.Hk = Hk;
    a.sign = 1.f;
    a.cu = cu_seqlens;
    a.kv_lens = kv_lens;
    a.B = B;
    a.err = device_error_word();
    return launch<true>(name, a, spec->style, D, static_cast<cudaStream_t>(stream));
}
