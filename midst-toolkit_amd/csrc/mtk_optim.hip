// mtk_optim.hip — one AdamW step over many tensors.
//
//   m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in fp32 whatever p's type, rounded once.  Moments in 32 bits, or in 8: m and r = sqrt(v) as e4m3 codes under one power-of-two
// scale per 256 values of a tensor.  r rather than v because v spans twice the exponents: e4m3 holds r over 2^17.8, v over 2^35.
// The scale is the smallest power of two that keeps the block's largest value in range (448); being a power of two it moves
// seldom and exactly, so the grid the codes lie on stays put between steps.  A slow average moves by far less than half a code step
// per update (1 - b2 = 0.001 against steps of 1/8 to 1/16), so rounding to nearest would freeze it: a value goes up or down to a
// neighbouring code by a dither u instead, floor(y / step + u), where u = frac(i a + t phi) is a Weyl sequence over the value's
// place i in its tensor and the step count t - equidistributed over the steps for every value, exact over time, and reproducible
// without a generator's state.  A non-zero r never becomes 0 (it would divide a live m by eps): the smallest code stands in.
//
// Bound by bandwidth: 28 B a value with fp32 and 32-bit moments, 10 B with bf16 and 8-bit ones.  Up to 64 tensors ride in one launch's
// arguments (nothing to upload, nothing that a captured graph could find changed); a workgroup takes one chunk of one tensor.
// 55 million fp32 values in 192 tensors, 32-bit moments: 257 us (1.54 GB: 6.0 TB/s); 220 million bf16 values, 8-bit moments: 417 us (2.2 GB: 5.3 TB/s);
// 2.2 million fp32 values in 12 tensors: 11 us either way, from the caches.
#include <math.h>

#include "mtk_lowp.h"

namespace {

constexpr int MAXT = 64;       // tensors of a launch: 3.9 KB of kernel arguments
// Everything goes past the caches, both ways, where a step moves more than they hold: the next step would find nothing there.  us, past / through
// them: 55 million fp32 values with 32-bit moments 257 / 293, 220 million bf16 values with 8-bit ones 426 / 466.
constexpr int64_t kCaches = 256ll << 20;
constexpr int QB = 256;        // values that share a scale

struct AdamwHyper {
    float b1, c1, b2, c2;      // beta, 1 - beta
    float decay, step_size, inv_bc2, eps;
    uint32_t phase;            // t * phi, of the dither
};
struct AdamwArgs {
    void* p[MAXT];
    const void* g[MAXT];
    void* m[MAXT];
    void* v[MAXT];
    float* ms[MAXT];
    float* vs[MAXT];
    int64_t numel[MAXT];
    int32_t first[MAXT + 1];   // first chunk of a tensor; first[n] = chunks of the launch
    int n;
    bool nt;                   // past the caches
    AdamwHyper h;
    const AdamwHyper* dyn;     // read instead of h where given (a step whose count lives on the device): dyn[each * tensor]
    int each;                  // 1: every tensor has its own count, 0: one for all
};

constexpr uint32_t kPhi = 0x9E3779B1u, kPlaceM = 0x6A09E667u, kPlaceR = 0xBB67AE85u;

// exponent (unbiased) of the block scale of a largest magnitude with bits b > 0: the magnitude times 2^-k is in (224, 448]
__device__ __forceinline__ int scale_exp(uint32_t b) {
    const int k = (int)(b >> 23) - 135 + ((b & 0x7fffff) > 0x600000 ? 1 : 0);
    return k < -126 ? -126 : k;
}
__device__ __forceinline__ float pow2(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }

// |x| 2^-k rounded to the e4m3 neighbour that the dither w (its upper 20 bits) selects; exact in e4m3.  The dither is added to the 20 bits of the
// float behind e4m3's three and the sum cut: a carry is the step up.  Codes below 2^-6 are equally spaced, as those in [2^-6, 2^-5) are:
// such a value is moved there and back.
__device__ __forceinline__ float dither(float x, float inv_scale, uint32_t w, float lowest) {
    const float y = fabsf(x) * inv_scale;
    const float lift = y < 0x1p-6f ? 0x1p-6f : 0.f;
    const float q = __uint_as_float((__float_as_uint(y + lift) + (w >> 12)) & 0xfff00000u) - lift;
    return __builtin_amdgcn_fmed3f(q, lowest, 448.f);
}
// sqrt(v), correctly rounded but for rare ties, in six instructions: the hardware's reciprocal root and one correction.  The cap is the reciprocal
// root of the smallest normal number: it serves 0 and numbers below 2^-126 (counted as 0 by the instruction), whose roots stay small.  Of an
// infinity it makes NaN, which the rare path of the kernel looks after (220 million bf16 values 417 -> 420 us; by a select here 435).
__device__ __forceinline__ float fast_sqrt(float v) {
    const float y = fminf(__builtin_amdgcn_rsqf(v), 0x1p63f), r = v * y;
    return __builtin_fmaf(__builtin_fmaf(-r, r, v) * 0.5f, y, r);
}

template <int N> struct __attribute__((packed, aligned(1), may_alias)) CodeVec { uint32_t w[N / 4]; };
typedef uint32_t CodeWord __attribute__((aligned(1), may_alias));

template <int N> __device__ __forceinline__ void ld_codes(const uint8_t* p, int left, float* f, bool nt) {
    CodeVec<N> c;
    if (left >= N) {
        if (nt)
#pragma unroll
            for (int i = 0; i < N / 4; ++i) c.w[i] = __builtin_nontemporal_load(reinterpret_cast<const CodeWord*>(p) + i);
        else c = *reinterpret_cast<const CodeVec<N>*>(p);
    }
    else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            c.w[i] = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (4 * i + j < left) c.w[i] |= (uint32_t)p[4 * i + j] << (8 * j);
        }
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(c.w[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(c.w[i], true);
        f[4 * i] = lo[0]; f[4 * i + 1] = lo[1]; f[4 * i + 2] = hi[0]; f[4 * i + 3] = hi[1];
    }
}
template <int N> __device__ __forceinline__ void st_codes(uint8_t* p, int left, const float* q, bool nt) {
    CodeVec<N> c;
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i], q[4 * i + 1], 0, false);
        c.w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i + 2], q[4 * i + 3], w, true);
    }
    if (left >= N) {
        if (nt)
#pragma unroll
            for (int i = 0; i < N / 4; ++i) __builtin_nontemporal_store(c.w[i], reinterpret_cast<CodeWord*>(p) + i);
        else *reinterpret_cast<CodeVec<N>*>(p) = c;
    }
    else
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) p[i] = (uint8_t)(c.w[i / 4] >> (8 * (i & 3)));
}
template <int N> __device__ __forceinline__ void ld_f32(const float* p, int left, float* f, bool nt) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const mtk_vec<float> v = left - i < 4 ? mtk_ld_n(p + i, left - i) : nt ? mtk_ld_nt(p + i) : mtk_ld(p + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[i + j] = v.v[j];
    }
}
template <int N> __device__ __forceinline__ void st_f32(float* p, int left, const float* f, bool nt) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        mtk_vec<float> v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v.v[j] = f[i + j];
        if (left - i < 4) mtk_st_n(p + i, v, left - i);
        else if (nt) mtk_st_nt(p + i, v);
        else mtk_st(p + i, v);
    }
}

// A lane takes the V values of one 16-byte piece of p; 256 / V lanes (a wave with fp32, half a wave with 16 bits) hold a block of 256.
template <typename T, bool Q8>
__global__ __launch_bounds__(256) void k_adamw(AdamwArgs a) {
    constexpr int V = mtk_piece<T>::n, CH = 256 * V;  // values of a chunk: a multiple of QB
    const int b = blockIdx.x;
    int lo = 0, hi = a.n - 1;  // the tensor that holds chunk b: the last with first <= b
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.first[mid] <= b) lo = mid;
        else hi = mid - 1;
    }
    const AdamwHyper h = a.dyn ? a.dyn[lo * a.each] : a.h;
    const int64_t n = a.numel[lo], i0 = (int64_t)(b - a.first[lo]) * CH + (int64_t)threadIdx.x * V;
    const int left = n - i0 >= V ? V : (n > i0 ? (int)(n - i0) : 0);
    T* pp = (T*)a.p[lo] + i0;
    const T* gp = (const T*)a.g[lo] + i0;
    const bool nt = a.nt;
    const mtk_vec<T> p0 = left < V ? mtk_ld_n(pp, left) : nt ? mtk_ld_nt(pp) : mtk_ld(pp), g0 = left < V ? mtk_ld_n(gp, left) : nt ? mtk_ld_nt(gp) : mtk_ld(gp);
    float m[V], v[V];
    const int64_t blk = i0 / QB;
    if (Q8) {
        ld_codes<V>((const uint8_t*)a.m[lo] + i0, left, m, nt);
        ld_codes<V>((const uint8_t*)a.v[lo] + i0, left, v, nt);
        const float sm = left ? a.ms[lo][blk] : 0.f, sv = left ? a.vs[lo][blk] : 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            m[i] *= sm;
            v[i] *= sv;
            v[i] *= v[i];
        }
    } else {
        ld_f32<V>((const float*)a.m[lo] + i0, left, m, nt);
        ld_f32<V>((const float*)a.v[lo] + i0, left, v, nt);
    }
    mtk_vec<T> p1;
    float r[V];
    uint32_t am = 0, ar = 0;  // largest magnitudes, as bits: what is not finite comes out on top
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float g = (float)g0.v[i];
        m[i] = h.b1 * m[i] + h.c1 * g;
        v[i] = h.b2 * v[i] + h.c2 * (g * g);
        if (Q8) {  // bound by its instructions: the quotient by a reciprocal (one unit in its last place), the root as above
            r[i] = fast_sqrt(v[i]);
            p1.v[i] = (T)((float)p0.v[i] * h.decay - h.step_size * (m[i] * __builtin_amdgcn_rcpf(r[i] * h.inv_bc2 + h.eps)));
            const uint32_t bm = __float_as_uint(m[i]) & 0x7fffffffu, br = __float_as_uint(r[i]) & 0x7fffffffu;
            am = am > bm ? am : bm;
            ar = ar > br ? ar : br;
        } else {
            r[i] = sqrtf(v[i]);
            p1.v[i] = (T)((float)p0.v[i] * h.decay - h.step_size * (m[i] / (r[i] * h.inv_bc2 + h.eps)));
        }
    }
    auto store_p = [&]() {
        if (left < V) mtk_st_n(pp, p1, left);
        else if (nt) mtk_st_nt(pp, p1);
        else mtk_st(pp, p1);
    };
    if (!Q8) {
        store_p();
        st_f32<V>((float*)a.m[lo] + i0, left, m, nt);
        st_f32<V>((float*)a.v[lo] + i0, left, v, nt);
        return;
    }
    auto block_max = [](uint32_t a) {
#pragma unroll
        for (int d = 1; d < QB / V; d <<= 1) {
            const uint32_t o = (uint32_t)__shfl_xor((int)a, d);
            a = a > o ? a : o;
        }
        return a;
    };
    am = block_max(am);
    ar = block_max(ar);
    constexpr uint32_t kInf = 0x7f800000u;
    const bool bad = am >= kInf || ar >= kInf;  // the same in all lanes of a block
    if (__any(bad)) {  // rare: the scales go by the finite values (blocks without others keep theirs)
        // A mean square that overflowed (its root came out as NaN, though neither the gradient, which m would show, nor the old root is one): the
        // quotient is m / inf.  What was read is read again: kept for this, it would cost a quarter of the waves of a CU.
        float old[V];
        ld_codes<V>((const uint8_t*)a.v[lo] + i0, left, old, false);
        const mtk_vec<T> q0 = mtk_ld_n(pp, left);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (r[i] != r[i] && m[i] == m[i] && old[i] == old[i]) p1.v[i] = (T)((float)q0.v[i] * h.decay - h.step_size * (m[i] * 0.f));
        uint32_t fm = 0, fr = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const uint32_t bm = __float_as_uint(m[i]) & 0x7fffffffu, br = __float_as_uint(r[i]) & 0x7fffffffu;
            fm = bm < kInf && bm > fm ? bm : fm;
            fr = br < kInf && br > fr ? br : fr;
        }
        am = block_max(fm);
        ar = block_max(fr);
    }
    store_p();
    const int km = am ? scale_exp(am) : 0, kr = ar ? scale_exp(ar) : 0;
    const float im = pow2(-km), ir = pow2(-kr);
    uint32_t wm = (uint32_t)i0 * kPlaceM + h.phase, wr = (uint32_t)i0 * kPlaceR + h.phase;
    float qm[V], qr[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        qm[i] = copysignf(dither(m[i], im, wm, 0.f), m[i]);
        qr[i] = dither(r[i], ir, wr, r[i] > 0.f ? 0x1p-9f : 0.f);
        wm += kPlaceM;
        wr += kPlaceR;
    }
    if (bad) {  // infinities have no code: they and NaN become NaN, alone in their block
#pragma unroll
        for (int i = 0; i < V; ++i) {
            qm[i] = (__float_as_uint(m[i]) & 0x7fffffffu) < kInf ? qm[i] : __builtin_nanf("");
            qr[i] = (__float_as_uint(r[i]) & 0x7fffffffu) < kInf ? qr[i] : __builtin_nanf("");
        }
    }
    st_codes<V>((uint8_t*)a.m[lo] + i0, left, qm, nt);
    st_codes<V>((uint8_t*)a.v[lo] + i0, left, qr, nt);
    if (left && (threadIdx.x & (QB / V - 1)) == 0) {
        a.ms[lo][blk] = pow2(km);
        a.vs[lo][blk] = pow2(kr);
    }
}

__host__ __device__ inline AdamwHyper hyper(double lr, double b1, double b2, double eps, double wd, double t, uint32_t ti) {
    AdamwHyper h;
    h.b1 = (float)b1; h.c1 = (float)(1.0 - b1); h.b2 = (float)b2; h.c2 = (float)(1.0 - b2);
    h.decay = (float)(1.0 - lr * wd);
    h.step_size = (float)(lr / (1.0 - pow(b1, t)));
    h.inv_bc2 = 1.0f / (float)sqrt(1.0 - pow(b2, t));
    h.eps = (float)eps;
    h.phase = ti * kPhi;
    return h;
}

// Step counts on the device: counted up here, so a replayed graph's steps are its own.  A count belongs to a tensor (one may go without a gradient
// where its neighbours have theirs); a thread takes one.
constexpr int MAXC = 256;      // counts of a launch
struct CountArgs {
    int64_t* step[MAXC];
    int n;
};
__global__ __launch_bounds__(MAXC) void k_adamw_count(CountArgs a, const float* lr_dev, double lr, double b1, double b2, double eps, double wd, AdamwHyper* out) {
    const int i = threadIdx.x;
    if (i >= a.n) return;
    const int64_t t = *a.step[i] + 1;
    *a.step[i] = t;
    out[i] = hyper(lr_dev ? (double)*lr_dev : lr, b1, b2, eps, wd, (double)t, (uint32_t)t);
}

}  // namespace

extern "C" int64_t mtk_adamw_scales(int64_t numel) { return numel > 0 ? (numel + QB - 1) / QB : 0; }
extern "C" int64_t mtk_adamw_hyper_bytes(void) { return (int64_t)sizeof(AdamwHyper); }

extern "C" int mtk_adamw_count_each(int n_steps, int64_t* const* step, const float* lr_dev, double lr, double beta1, double beta2, double eps, double weight_decay,
                                    void* hyper_dev, mtk_stream stream) {
    if (n_steps < 0 || (n_steps > 0 && (!step || !hyper_dev))) MTK_FAIL(MTK_ERR_ARG, "mtk_adamw_count: null pointer or negative count");
    if (!(lr_dev || lr >= 0) || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0) || !(weight_decay >= 0))
        MTK_FAIL(MTK_ERR_ARG, "mtk_adamw_count: lr %g, betas %g %g, eps %g, weight_decay %g", lr, beta1, beta2, eps, weight_decay);
    for (int i = 0; i < n_steps; ++i)
        if (!step[i]) MTK_FAIL(MTK_ERR_ARG, "mtk_adamw_count: step %d: null pointer", i);
    for (int i = 0; i < n_steps; i += MAXC) {
        CountArgs a;
        a.n = n_steps - i < MAXC ? n_steps - i : MAXC;
        for (int j = 0; j < a.n; ++j) a.step[j] = step[i + j];
        k_adamw_count<<<1, MAXC, 0, (hipStream_t)stream>>>(a, lr_dev, lr, beta1, beta2, eps, weight_decay, (AdamwHyper*)hyper_dev + i);
    }
    MTK_HIP(hipGetLastError());
    return MTK_OK;
}
extern "C" int mtk_adamw_count(int64_t* step, const float* lr_dev, double lr, double beta1, double beta2, double eps, double weight_decay,
                               void* hyper_dev, mtk_stream stream) {
    return mtk_adamw_count_each(1, &step, lr_dev, lr, beta1, beta2, eps, weight_decay, hyper_dev, stream);
}

static int adamw_step(int n_tensors, void* const* p, const void* const* g, void* const* m, void* const* v, float* const* m_scale, float* const* v_scale,
                      const int64_t* numel, int dtype, int state_bits, double lr, double beta1, double beta2, double eps, double weight_decay, int64_t step,
                      const void* hyper_dev, int each, mtk_stream stream) {
    if (n_tensors < 0 || (n_tensors > 0 && (!p || !g || !m || !v || !numel))) MTK_FAIL(MTK_ERR_ARG, "mtk_adamw_step: null pointer or negative count");
    if (!mtk_dtype_ok(dtype)) MTK_FAIL(MTK_ERR_UNSUPPORTED, "mtk_adamw_step: dtype %d", dtype);
    if (state_bits != 32 && state_bits != 8) MTK_FAIL(MTK_ERR_UNSUPPORTED, "mtk_adamw_step: moments in %d bits (8 or 32)", state_bits);
    if (state_bits == 8 && n_tensors > 0 && (!m_scale || !v_scale)) MTK_FAIL(MTK_ERR_ARG, "mtk_adamw_step: 8-bit moments need their scales");
    if (!(lr >= 0) || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0) || !(weight_decay >= 0))
        MTK_FAIL(MTK_ERR_ARG, "mtk_adamw_step: lr %g, betas %g %g, eps %g, weight_decay %g", lr, beta1, beta2, eps, weight_decay);
    if (!hyper_dev && step < 1) MTK_FAIL(MTK_ERR_ARG, "mtk_adamw_step: step %lld (the first is 1)", (long long)step);
    const int64_t chunk = 256 * (16 / mtk_dtype_size(dtype));
    for (int i = 0; i < n_tensors; ++i) {
        if (numel[i] < 0) MTK_FAIL(MTK_ERR_ARG, "mtk_adamw_step: tensor %d has %lld values", i, (long long)numel[i]);
        if (numel[i] == 0) continue;
        if (!p[i] || !g[i] || !m[i] || !v[i] || (state_bits == 8 && (!m_scale[i] || !v_scale[i]))) MTK_FAIL(MTK_ERR_ARG, "mtk_adamw_step: tensor %d: null pointer", i);
        if (numel[i] / chunk >= (1 << 23)) MTK_FAIL(MTK_ERR_UNSUPPORTED, "mtk_adamw_step: tensor %d has %lld values", i, (long long)numel[i]);
    }
    AdamwArgs a;
    int64_t bytes = 0;
    for (int i = 0; i < n_tensors; ++i) bytes += numel[i] * (3 * mtk_dtype_size(dtype) + (state_bits == 8 ? 4 : 16));
    a.nt = bytes > kCaches;
    if (!hyper_dev) a.h = hyper(lr, beta1, beta2, eps, weight_decay, (double)step, (uint32_t)step);
    a.each = each;
    int i = 0;
    while (i < n_tensors) {
        a.n = 0;
        a.dyn = hyper_dev ? (const AdamwHyper*)hyper_dev + (each ? i : 0) : nullptr;
        int64_t chunks = 0;
        for (; i < n_tensors && a.n < MAXT; ++i) {  // an empty tensor has no chunk, but its place among the counts
            const int64_t c = (numel[i] + chunk - 1) / chunk;
            if (chunks + c >= (1 << 24)) break;  // a launch holds fewer than 2^32 threads
            a.p[a.n] = p[i]; a.g[a.n] = g[i]; a.m[a.n] = m[i]; a.v[a.n] = v[i];
            a.ms[a.n] = state_bits == 8 ? m_scale[i] : nullptr;
            a.vs[a.n] = state_bits == 8 ? v_scale[i] : nullptr;
            a.numel[a.n] = numel[i];
            a.first[a.n++] = (int32_t)chunks;
            chunks += c;
        }
        if (chunks == 0) continue;
        a.first[a.n] = (int32_t)chunks;
        mtk_by_type(dtype, [&](auto t) {
            typedef decltype(t) T;
            if (state_bits == 8) k_adamw<T, true><<<(unsigned)chunks, 256, 0, (hipStream_t)stream>>>(a);
            else k_adamw<T, false><<<(unsigned)chunks, 256, 0, (hipStream_t)stream>>>(a);
        });
    }
    MTK_HIP(hipGetLastError());
    return MTK_OK;
}

extern "C" int mtk_adamw_step(int n_tensors, void* const* p, const void* const* g, void* const* m, void* const* v, float* const* m_scale,
                              float* const* v_scale, const int64_t* numel, int dtype, int state_bits, double lr, double beta1, double beta2,
                              double eps, double weight_decay, int64_t step, const void* hyper_dev, mtk_stream stream) {
    return adamw_step(n_tensors, p, g, m, v, m_scale, v_scale, numel, dtype, state_bits, lr, beta1, beta2, eps, weight_decay, step, hyper_dev, 0, stream);
}
extern "C" int mtk_adamw_step_each(int n_tensors, void* const* p, const void* const* g, void* const* m, void* const* v, float* const* m_scale, float* const* v_scale,
                                   const int64_t* numel, int dtype, int state_bits, const void* hyper_dev, mtk_stream stream) {
    if (n_tensors > 0 && !hyper_dev) MTK_FAIL(MTK_ERR_ARG, "mtk_adamw_step: null pointer or negative count");
    return adamw_step(n_tensors, p, g, m, v, m_scale, v_scale, numel, dtype, state_bits, 0.0, 0.0, 0.0, 0.0, 0.0, 1, hyper_dev, 1, stream);
}
