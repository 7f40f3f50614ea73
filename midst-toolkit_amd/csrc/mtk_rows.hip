// mtk_rows.hip — (record, model) pairs sorted by model and back.
//
// A pair is an entry of index[n][k] (model of record n's copy k).  Plan: key = index, or n_groups for a pair without a model (-1, or
// out of range); order = stable argsort(key), slot = its inverse, offsets[e] = number of pairs with key < e.
//   dispatch  xs[s] = x[order[s] / k] (times w[order[s]])      combine  out[n] = sum_j w[n, j] y[slot[n, j]]
// and each is the other's gradient, so two row kernels serve the four directions; the gradient of the weights, <gout[n], y[s]>, rides
// in the dispatch of gout.  Sums run over j (or along the row in a fixed tree) in fp32: no atomics, the same bits every run.
#include "mtk_lowp.h"

namespace {

constexpr int RT = 512, RW = RT / 64;      // threads / waves of a routing workgroup
constexpr int64_t kRouteChunk = 8192;      // pairs of a workgroup, until there are kRouteBlocks of them
constexpr int kRouteBlocks = 128;

struct RouteArgs {
    const int64_t* index;
    int64_t P;        // pairs
    int E, nblk;
    int64_t chunk;    // pairs per workgroup, a multiple of RT
    int32_t *order, *slot, *offsets, *counts;  // counts [nblk][E + 1], for nblk > 1
};

__device__ __forceinline__ int route_key(int64_t v, int E) { return v >= 0 && v < E ? (int)v : E; }

// counts of one workgroup's pairs per key (integer LDS atomics: any order gives the same counts)
__global__ __launch_bounds__(RT) void k_route_count(RouteArgs a) {
    extern __shared__ int32_t sm[];
    const int bins = a.E + 1;
    for (int i = threadIdx.x; i < bins; i += RT) sm[i] = 0;
    __syncthreads();
    const int64_t lo = blockIdx.x * a.chunk, hi = lo + a.chunk < a.P ? lo + a.chunk : a.P;
    for (int64_t i = lo + threadIdx.x; i < hi; i += RT) atomicAdd(&sm[route_key(a.index[i], a.E)], 1);
    __syncthreads();
    for (int i = threadIdx.x; i < bins; i += RT) a.counts[(int64_t)blockIdx.x * bins + i] = sm[i];
}

// Stable placement.  A wave owns a contiguous part of its workgroup's pairs: counts per (wave, key), a prefix over keys, earlier
// workgroups and earlier waves, then 64 pairs at a time: the lanes with the same key find each other by one ballot per key bit,
// a lane's place is the wave's running counter plus the equal lanes below it.
__global__ __launch_bounds__(RT) void k_route_place(RouteArgs a) {
    extern __shared__ int32_t sm[];
    const int bins = a.E + 1, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int32_t* ctr = sm;                    // [RW][bins]
    int32_t* base = sm + RW * bins;       // [bins] first slot of this workgroup's pairs of a key
    int32_t* tot = base + bins;           // [bins] totals, then their exclusive prefix
    for (int i = tid; i < RW * bins; i += RT) ctr[i] = 0;
    __syncthreads();
    const int64_t lo = blockIdx.x * a.chunk, hi = lo + a.chunk < a.P ? lo + a.chunk : a.P;
    const int64_t per = a.chunk / RW, wlo = lo + wave * per, whi = wlo + per < hi ? wlo + per : hi;
    for (int64_t i = wlo + lane; i < whi; i += 64) atomicAdd(&ctr[wave * bins + route_key(a.index[i], a.E)], 1);
    __syncthreads();
    for (int b = tid; b < bins; b += RT) {
        int before = 0, all = 0;
        if (a.nblk > 1) {
            for (int q = 0; q < a.nblk; ++q) {
                const int c = a.counts[(int64_t)q * bins + b];
                before += q < (int)blockIdx.x ? c : 0;
                all += c;
            }
        } else {
            for (int w = 0; w < RW; ++w) all += ctr[w * bins + b];
        }
        base[b] = before;
        tot[b] = all;
    }
    __syncthreads();
    // exclusive prefix over the keys: a wave scans 64 at a time, carrying the sum (at most 17 rounds)
    if (wave == 0) {
        int carry = 0;
        for (int b0 = 0; b0 < bins; b0 += 64) {
            const int b = b0 + lane, v = b < bins ? tot[b] : 0;
            int s = v;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int t = __shfl_up(s, d);
                if (lane >= d) s += t;
            }
            if (b < bins) tot[b] = carry + s - v;
            carry += __shfl(s, 63);
        }
    }
    __syncthreads();
    for (int b = tid; b < bins; b += RT) {
        if (blockIdx.x == 0) a.offsets[b] = tot[b];  // offsets[E] = the number of pairs with a model
        int at = tot[b] + base[b];
        for (int w = 0; w < RW; ++w) {
            const int c = ctr[w * bins + b];
            ctr[w * bins + b] = at;
            at += c;
        }
    }
    __syncthreads();
    int bits = 0;
    while ((1 << bits) < bins) ++bits;
    volatile int32_t* my = ctr + wave * bins;  // one wave's LDS operations complete in order: no barrier inside the loop
    for (int64_t i0 = wlo; i0 < whi; i0 += 64) {
        const int64_t i = i0 + lane;
        const bool live = i < whi;
        const int64_t v = live ? a.index[i] : -1;
        const int key = route_key(v, a.E);
        unsigned long long same = __ballot(live);
        for (int b = 0; b < bits; ++b) {
            const unsigned long long m = __ballot((key >> b) & 1);
            same &= ((key >> b) & 1) ? m : ~m;
        }
        const unsigned long long below = same & ((1ull << lane) - 1);
        if (live) {
            const int s = my[key] + __popcll(below);
            a.slot[i] = s;
            a.order[s] = v < -1 || v >= a.E ? ~(int32_t)i : (int32_t)i;
            if (below == 0) my[key] = s + __popcll(same);
        }
    }
}

struct RowsArgs {
    int64_t n;        // rows written
    int64_t other;    // rows of the tensor that is read
    int64_t D, ld;    // width; row stride of the tensor that is read
    int k;            // copies per record
    const int32_t* map;  // order [n] (dispatch) or slot [n][k] (combine)
    const float* w;      // [pairs] or null
    int lpr;             // lanes of a row: a power of two up to 64
};

// xs[s] = x[pair / k] (times w[pair]); pair = order[s].  A row of a pair whose index was out of range (stored as ~pair) is NaN: loud,
// never an out-of-range read.  With y: dw[pair] = <x[pair / k], y[s]> as well (x is the gradient of the combined rows then).
// Bound by bandwidth: a row belongs to lpr lanes, each moving 16-byte pieces, so a wave reads whole lines.
template <typename T, bool W, bool DOT>
__global__ __launch_bounds__(256) void k_dispatch(RowsArgs a, const T* __restrict__ x, T* __restrict__ xs, const T* __restrict__ y, float* __restrict__ dw) {
    constexpr int V = mtk_piece<T>::n;
    const int sub = threadIdx.x & (a.lpr - 1);
    for (int64_t s = (int64_t)blockIdx.x * (256 / a.lpr) + threadIdx.x / a.lpr; s < a.n; s += (int64_t)gridDim.x * (256 / a.lpr)) {
        float dot = 0.f;
        int p = a.map[s];
        const bool bad = p < 0;
        p = bad ? ~p : p;
        int64_t row = p / a.k;
        row = row < a.other ? row : a.other - 1;
        const float w = bad ? __builtin_nanf("") : (W ? a.w[p] : 1.f);
        const T* src = x + row * a.ld;
        T* dst = xs ? xs + s * a.D : nullptr;
        const T* ys = DOT ? y + s * a.D : nullptr;
        for (int64_t c = (int64_t)sub * V; c < a.D; c += (int64_t)a.lpr * V) {
            const int left = a.D - c < V ? (int)(a.D - c) : V;
            mtk_vec<T> v = left == V ? mtk_ld(src + c) : mtk_ld_n(src + c, left);
            if (DOT) {
                const mtk_vec<T> q = left == V ? mtk_ld(ys + c) : mtk_ld_n(ys + c, left);
#pragma unroll
                for (int i = 0; i < V; ++i) dot += (float)v.v[i] * (float)q.v[i];
            }
            if (W || bad) {
#pragma unroll
                for (int i = 0; i < V; ++i) v.v[i] = (T)((float)v.v[i] * w);
            }
            if (!DOT || dst) {
                if (left == V) mtk_st(dst + c, v);
                else mtk_st_n(dst + c, v, left);
            }
        }
        if (DOT) {  // the lanes of a row leave the loop together, and the exchange stays among them
            for (int d = a.lpr >> 1; d > 0; d >>= 1) dot += __shfl_xor(dot, d);
            if (sub == 0) dw[p] = dot;
        }
    }
}

// out[n] = sum_j (w[n, j]) y[slot[n, j]], j ascending, fp32, rounded once
template <typename T, bool W>
__global__ __launch_bounds__(256) void k_combine(RowsArgs a, const T* __restrict__ y, T* __restrict__ out) {
    constexpr int V = mtk_piece<T>::n;
    const int sub = threadIdx.x & (a.lpr - 1);
    for (int64_t n = (int64_t)blockIdx.x * (256 / a.lpr) + threadIdx.x / a.lpr; n < a.n; n += (int64_t)gridDim.x * (256 / a.lpr))
    for (int64_t c = (int64_t)sub * V; c < a.D; c += (int64_t)a.lpr * V) {
        const int32_t* slots = a.map + n * a.k;
        const float* ws = W ? a.w + n * a.k : nullptr;
        const int left = a.D - c < V ? (int)(a.D - c) : V;
        float acc[V];
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.f;
        for (int j = 0; j < a.k; ++j) {
            int64_t s = slots[j];
            s = s < 0 ? 0 : (s < a.other ? s : a.other - 1);
            const float w = W ? ws[j] : 1.f;
            const T* src = y + s * a.ld + c;
            const mtk_vec<T> v = left == V ? mtk_ld(src) : mtk_ld_n(src, left);
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += W ? w * (float)v.v[i] : (float)v.v[i];
        }
        mtk_vec<T> o;
#pragma unroll
        for (int i = 0; i < V; ++i) o.v[i] = (T)acc[i];
        if (left == V) mtk_st(out + n * a.D + c, o);
        else mtk_st_n(out + n * a.D + c, o, left);
    }
}

int lanes_per_row(int64_t D, int V) {
    int l = 1;
    while (l < 64 && (int64_t)l * V < D) l <<= 1;
    return l;
}

// one row per lane group, up to 2^22 workgroups (a launch holds fewer than 2^32 threads)
unsigned rows_grid(const RowsArgs& a) {
    const int64_t nb = (a.n + 256 / a.lpr - 1) / (256 / a.lpr);
    return (unsigned)(nb < (1 << 22) ? nb : (1 << 22));
}

int route_blocks(int64_t P, int64_t* chunk) {
    const int64_t nb = P < kRouteChunk ? 1 : (P + kRouteChunk - 1) / kRouteChunk;
    const int64_t nblk = nb < kRouteBlocks ? nb : kRouteBlocks;
    *chunk = mtk_up((P + nblk - 1) / nblk, RT);
    return (int)((P + *chunk - 1) / *chunk);
}

int rows_check(const char* who, int64_t n, int k, int64_t D, int64_t ld, int dtype) {
    if (n < 0 || k < 1 || D < 1 || ld < 0) MTK_FAIL(MTK_ERR_ARG, "%s: bad sizes (rows %lld, copies %d, width %lld)", who, (long long)n, k, (long long)D);
    if (n > 0x7fffffffll / k) MTK_FAIL(MTK_ERR_UNSUPPORTED, "%s: %lld rows of %d copies exceed 2^31 - 1 pairs", who, (long long)n, k);
    if (!mtk_dtype_ok(dtype)) MTK_FAIL(MTK_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
    return MTK_OK;
}

}  // namespace

extern "C" int64_t mtk_route_rows_work(int64_t n_pairs, int n_groups) {
    if (n_pairs < 1 || n_groups < 1) return 0;
    int64_t chunk;
    const int nblk = route_blocks(n_pairs, &chunk);
    return nblk > 1 ? (int64_t)nblk * (n_groups + 1) : 0;
}

extern "C" int mtk_route_rows(int64_t n_pairs, const int64_t* index, int n_groups, int32_t* order, int32_t* slot, int32_t* offsets,
                              int32_t* work, int64_t work_elems, mtk_stream stream) {
    if (n_pairs < 0 || !offsets || (n_pairs > 0 && (!index || !order || !slot))) MTK_FAIL(MTK_ERR_ARG, "mtk_route_rows: null pointer or negative count");
    if (n_groups < 1 || n_groups > MTK_ROUTE_MAX_GROUPS) MTK_FAIL(MTK_ERR_UNSUPPORTED, "mtk_route_rows: %d groups (1 to %d)", n_groups, MTK_ROUTE_MAX_GROUPS);
    if (n_pairs > 0x7fffffffll) MTK_FAIL(MTK_ERR_UNSUPPORTED, "mtk_route_rows: %lld pairs exceed 2^31 - 1", (long long)n_pairs);
    RouteArgs a{index, n_pairs, n_groups, 1, RT, order, slot, offsets, work};
    if (n_pairs > 0) a.nblk = route_blocks(n_pairs, &a.chunk);
    const int bins = n_groups + 1;
    const hipStream_t s = (hipStream_t)stream;
    if (a.nblk > 1) {
        if (!work || work_elems < (int64_t)a.nblk * bins) MTK_FAIL(MTK_ERR_ARG, "mtk_route_rows: workspace of %lld elements, %lld needed", (long long)work_elems, (long long)a.nblk * bins);
        k_route_count<<<a.nblk, RT, bins * sizeof(int32_t), s>>>(a);
    }
    k_route_place<<<a.nblk, RT, (size_t)(RW * bins + 2 * bins) * sizeof(int32_t), s>>>(a);
    MTK_HIP(hipGetLastError());
    return MTK_OK;
}

extern "C" int mtk_rows_dispatch(int64_t n_rows, int k, int64_t D, int dtype, const void* x, int64_t x_ld, const int32_t* order, const float* w,
                                 void* xs, const void* y, float* dw, mtk_stream stream) {
    if (const int rc = rows_check("mtk_rows_dispatch", n_rows, k, D, x_ld, dtype)) return rc;
    if (n_rows == 0) return MTK_OK;
    if (!x || !order || (!xs && !dw) || ((y != nullptr) != (dw != nullptr))) MTK_FAIL(MTK_ERR_ARG, "mtk_rows_dispatch: null pointer");
    mtk_by_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        RowsArgs a{n_rows * k, n_rows, D, x_ld, k, order, w, lanes_per_row(D, mtk_piece<T>::n)};
        const unsigned grid = rows_grid(a);
        const T* xp = (const T*)x;
        if (dw) {
            if (w) k_dispatch<T, true, true><<<grid, 256, 0, (hipStream_t)stream>>>(a, xp, (T*)xs, (const T*)y, dw);
            else k_dispatch<T, false, true><<<grid, 256, 0, (hipStream_t)stream>>>(a, xp, (T*)xs, (const T*)y, dw);
        } else {
            if (w) k_dispatch<T, true, false><<<grid, 256, 0, (hipStream_t)stream>>>(a, xp, (T*)xs, nullptr, nullptr);
            else k_dispatch<T, false, false><<<grid, 256, 0, (hipStream_t)stream>>>(a, xp, (T*)xs, nullptr, nullptr);
        }
    });
    MTK_HIP(hipGetLastError());
    return MTK_OK;
}

extern "C" int mtk_rows_combine(int64_t n_rows, int k, int64_t D, int dtype, const void* y, int64_t y_ld, const int32_t* slot, const float* w,
                                void* out, mtk_stream stream) {
    if (const int rc = rows_check("mtk_rows_combine", n_rows, k, D, y_ld, dtype)) return rc;
    if (n_rows == 0) return MTK_OK;
    if (!y || !slot || !out) MTK_FAIL(MTK_ERR_ARG, "mtk_rows_combine: null pointer");
    mtk_by_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        RowsArgs a{n_rows, n_rows * k, D, y_ld, k, slot, w, lanes_per_row(D, mtk_piece<T>::n)};
        const unsigned grid = rows_grid(a);
        if (w) k_combine<T, true><<<grid, 256, 0, (hipStream_t)stream>>>(a, (const T*)y, (T*)out);
        else k_combine<T, false><<<grid, 256, 0, (hipStream_t)stream>>>(a, (const T*)y, (T*)out);
    });
    MTK_HIP(hipGetLastError());
    return MTK_OK;
}
