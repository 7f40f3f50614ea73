// mtk_rows.hip — (record, model) pairs sorted by model and back.
//
// A pair is an entry of index[n][k] (model of record n's copy k).  Plan: key = index, or n_groups for a pair without a model (-1, or
// out of range); order = stable argsort(key), slot = its inverse, offsets[e] = number of pairs with key < e.
//   dispatch  xs[s] = x[order[s] / k] (times w[order[s]])      combine  out[n] = sum_j w[n, j] y[slot[n, j]]
// and each is the other's gradient, so two row kernels serve the four directions; the gradient of the weights, <gout[n], y[s]>, rides
// in the dispatch of gout.  Sums run over j (or along the row in a fixed tree) in fp32: no atomics, the same bits every run.
#include <type_traits>

#include "mtk_lowp.h"

namespace {

constexpr int RT = 512, RW = RT / 64;      // threads / waves of a routing workgroup
constexpr int64_t kRouteChunk = 2048;      // pairs of a workgroup, until there are kRouteBlocks of them
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
// a lane's place is the wave's running counter plus the equal lanes below it.  Bound by latency: 48 pairs 2.8 us (one workgroup, one launch),
// 16,396 pairs 10 us and 200,000 pairs 12 us with the counts.
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
    for (int b = tid; b < bins; b += RT) base[b] = tot[b] = 0;
    __syncthreads();
    if (a.nblk > 1) {
        for (int i = tid; i < a.nblk * bins; i += RT) {
            const int q = i / bins, b = i - q * bins, c = a.counts[i];
            if (c) {
                atomicAdd(&tot[b], c);
                if (q < (int)blockIdx.x) atomicAdd(&base[b], c);
            }
        }
    } else {
        for (int i = tid; i < RW * bins; i += RT)
            if (ctr[i]) atomicAdd(&tot[i % bins], ctr[i]);
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
    int64_t ahead = wlo + lane < whi ? a.index[wlo + lane] : -1;
    for (int64_t i0 = wlo; i0 < whi; i0 += 64) {
        const int64_t i = i0 + lane;
        const bool live = i < whi;
        const int64_t v = ahead;
        ahead = i + 64 < whi ? a.index[i + 64] : -1;
        const int key = route_key(v, a.E);
        unsigned long long same = __ballot(live);
        for (int b = 0; b < bits; ++b) {
            const unsigned long long m = __ballot((key >> b) & 1);
            same &= ((key >> b) & 1) ? m : ~m;
        }
        const unsigned long long below = same & ((1ull << lane) - 1);
        if (live) {
            const int s = my[key] + __popcll(below);
            const bool bad = v < -1 || v >= a.E;
            a.slot[i] = bad ? ~s : s;
            a.order[s] = bad ? ~(int32_t)i : (int32_t)i;
            if (below == 0) my[key] = s + __popcll(same);
        }
    }
}

struct RowsArgs {
    int64_t n;        // records
    int64_t other;    // pairs
    int64_t D, ld;    // width; row stride of the tensor that is read
    int k;            // copies per record
    const int32_t* map;  // slot [n][k]
    const float* w;      // [pairs] or null
    int lpr;             // lanes of a row: a power of two up to 64
    bool nt;             // past the caches
};

// A pair whose index was out of range has ~place for a slot: its rows are NaN on both ways, loud, and never an out-of-range access.
// KC: copies at a time, 1, 2 or 4.
template <int KC> struct Copies {
    int32_t s[KC];
    float w[KC];
};
// the slots and weights of record n's copies j0 ..; behind the last copy, the first again.  Loaded a record ahead of their use: they would
// otherwise be a round trip to memory in front of every row.
template <bool W, int KC> __device__ __forceinline__ Copies<KC> copies_of(const RowsArgs& a, int64_t n, int j0) {
    Copies<KC> c;
    n = n < a.n ? n : a.n - 1;
#pragma unroll
    for (int j = 0; j < KC; ++j) {
        const int64_t pair = n * a.k + (j0 + j < a.k ? j0 + j : j0);
        c.s[j] = a.map[pair];
        c.w[j] = W ? a.w[pair] : 1.f;
    }
    return c;
}
__device__ __forceinline__ int64_t place_of(int32_t s, int64_t pairs, bool& bad) {
    bad = s < 0;
    s = bad ? ~s : s;
    return s < pairs ? s : pairs - 1;
}

// A row's last piece, where it is not whole, starts earlier and brings some elements a second time: the same values are written twice, and a dot product
// skips what the lane before has.  (Loads and stores of single elements instead cost every row a second pass through the loop's
// body; only rows narrower than a piece have them.)
//
// xs[slot[n, j]] = x[n] (times w[n, j]) for all copies j: a record's row is read once and written k times.  With y: dw[n, j] =
// <x[n], y[slot[n, j]]> as well (x is the gradient of the combined rows then).  Bound by bandwidth: a row belongs to lpr lanes, each moving
// 16-byte pieces, so a wave touches whole lines.  4,099 rows of 1,021 fp32 in four copies (84 MB): 20 us, with the weights' gradient
// (151 MB) 30 us; 24 rows of 120: 2.7 us, a launch.
template <typename T, bool W, bool DOT, int KC>
__global__ __launch_bounds__(256) void k_dispatch(RowsArgs a, const T* __restrict__ x, T* __restrict__ xs, const T* __restrict__ y, float* __restrict__ dw) {
    constexpr int V = mtk_piece<T>::n;
    const int sub = threadIdx.x & (a.lpr - 1);
    const int64_t pairs = a.n * a.k, stride = (int64_t)gridDim.x * (256 / a.lpr);
    int64_t n = (int64_t)blockIdx.x * (256 / a.lpr) + threadIdx.x / a.lpr;
    Copies<KC> next = copies_of<W, KC>(a, n, 0);
    for (; n < a.n; n += stride) {
        const T* src = x + n * a.ld;
        for (int j0 = 0; j0 < a.k; j0 += KC) {
            const int nj = a.k - j0 < KC ? a.k - j0 : KC;
            const Copies<KC> cur = next;
            next = j0 + KC < a.k ? copies_of<W, KC>(a, n, j0 + KC) : copies_of<W, KC>(a, n + stride, 0);
            int64_t at[KC];
            float w[KC], dot[KC];
            bool scaled = W;
#pragma unroll
            for (int j = 0; j < KC; ++j) {
                bool bad;
                at[j] = place_of(cur.s[j], pairs, bad) * a.D;
                w[j] = bad ? __builtin_nanf("") : cur.w[j];
                scaled |= bad;
                dot[j] = 0.f;
            }
#pragma unroll 2
            for (int64_t c0 = (int64_t)sub * V; c0 < a.D; c0 += (int64_t)a.lpr * V) {
                const int64_t c = c0 + V <= a.D || a.D < V ? c0 : a.D - V;
                const int left = a.D < V ? (int)a.D : V, first = (int)(c0 - c);
                const mtk_vec<T> v = left < V ? mtk_ld_n(src + c, left) : a.nt ? mtk_ld_nt(src + c) : mtk_ld(src + c);
                if (DOT) {
#pragma unroll
                    for (int j = 0; j < KC; ++j) {
                        if (j >= nj) break;
                        const T* ys = y + at[j] + c;
                        const mtk_vec<T> q = left < V ? mtk_ld_n(ys, left) : a.nt ? mtk_ld_nt(ys) : mtk_ld(ys);
#pragma unroll
                        for (int i = 0; i < V; ++i) dot[j] += i >= first ? (float)v.v[i] * (float)q.v[i] : 0.f;
                    }
                }
                if (!DOT || xs) {
#pragma unroll
                    for (int j = 0; j < KC; ++j) {
                        if (j >= nj) break;
                        mtk_vec<T> o = v;
                        if (scaled) {
#pragma unroll
                            for (int i = 0; i < V; ++i) o.v[i] = (T)((float)v.v[i] * w[j]);
                        }
                        T* op = xs + at[j] + c;
                        if (left < V) mtk_st_n(op, o, left);
                        else if (a.nt) mtk_st_nt(op, o);
                        else mtk_st(op, o);
                    }
                }
            }
            if (DOT) {  // the lanes of a row leave the loop together, and the exchange stays among them
#pragma unroll
                for (int j = 0; j < KC; ++j) {
                    for (int d = a.lpr >> 1; d > 0; d >>= 1) dot[j] += __shfl_xor(dot[j], d);
                    if (sub == 0 && j < nj) dw[n * a.k + j0 + j] = dot[j];
                }
            }
        }
    }
}

// out[n] = sum_j (w[n, j]) y[slot[n, j]], j ascending, fp32, rounded once; four copies' loads in flight.  4,099 rows of 1,021 fp32 from four copies
// each (84 MB): 15 us weighted, with the rows still in the caches, 25 us when not.
template <typename T, bool W, int KC>
__global__ __launch_bounds__(256) void k_combine(RowsArgs a, const T* __restrict__ y, T* __restrict__ out) {
    constexpr int V = mtk_piece<T>::n;
    const int sub = threadIdx.x & (a.lpr - 1);
    const int64_t stride = (int64_t)gridDim.x * (256 / a.lpr);
    int64_t n = (int64_t)blockIdx.x * (256 / a.lpr) + threadIdx.x / a.lpr;
    Copies<KC> next = copies_of<W, KC>(a, n, 0);
    for (; n < a.n; n += stride) {
        const Copies<KC> first = next;
        next = copies_of<W, KC>(a, n + stride, 0);
#pragma unroll 2
        for (int64_t c0 = (int64_t)sub * V; c0 < a.D; c0 += (int64_t)a.lpr * V) {
            const int64_t c = c0 + V <= a.D || a.D < V ? c0 : a.D - V;
            const int left = a.D < V ? (int)a.D : V;
            float acc[V];
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = 0.f;
            auto add = [&](const Copies<KC>& cp, int nj) {
                mtk_vec<T> v[KC];
                float w[KC];
#pragma unroll
                for (int j = 0; j < KC; ++j) {
                    if (j >= nj) break;
                    bool bad;
                    const T* src = y + place_of(cp.s[j], a.other, bad) * a.ld + c;
                    w[j] = bad ? __builtin_nanf("") : cp.w[j];
                    v[j] = left < V ? mtk_ld_n(src, left) : a.nt ? mtk_ld_nt(src) : mtk_ld(src);
                }
#pragma unroll
                for (int j = 0; j < KC; ++j) {
                    if (j >= nj) break;
#pragma unroll
                    for (int i = 0; i < V; ++i) acc[i] += w[j] * (float)v[j].v[i];
                }
            };
            add(first, a.k < KC ? a.k : KC);
            for (int j0 = KC; j0 < a.k; j0 += KC) add(copies_of<W, KC>(a, n, j0), a.k - j0 < KC ? a.k - j0 : KC);
            mtk_vec<T> o;
#pragma unroll
            for (int i = 0; i < V; ++i) o.v[i] = (T)acc[i];
            T* op = out + n * a.D + c;
            if (left < V) mtk_st_n(op, o, left);
            else if (a.nt) mtk_st_nt(op, o);
            else mtk_st(op, o);
        }
    }
}

int lanes_per_row(int64_t D, int V) {
    int l = 1;
    while (l < 64 && (int64_t)l * V < D) l <<= 1;
    return l;
}

// Rows go past the caches, read and written, where what a call moves exceeds what they hold (256 MB): the result's readers would find nothing
// there.  us, 100,000 rows of 1024 bf16, two copies, past them / reads through them / all through them: dispatch 117 / 115 / 221, weighted combine
// 131 / 158, dispatch with the weights' gradient 204 / 270 (1.0 GB: 5.0 TB/s, past what a large copy reaches).
constexpr int64_t kCaches = 256ll << 20;
template <typename F> void by_flags(bool a, bool b, int k, F f) {
    auto third = [&](auto ta, auto tb) {
        if (k == 1) f(ta, tb, std::integral_constant<int, 1>());
        else if (k == 2) f(ta, tb, std::integral_constant<int, 2>());
        else f(ta, tb, std::integral_constant<int, 4>());
    };
    auto second = [&](auto ta) { b ? third(ta, std::true_type()) : third(ta, std::false_type()); };
    a ? second(std::true_type()) : second(std::false_type());
}

// a row per lane group; from 16 workgroups a CU on they walk
unsigned rows_grid(const RowsArgs& a) {
    const int64_t nb = (a.n + 256 / a.lpr - 1) / (256 / a.lpr);
    return (unsigned)(nb < 4096 ? nb : 4096);
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

extern "C" int mtk_rows_dispatch(int64_t n_rows, int k, int64_t D, int dtype, const void* x, int64_t x_ld, const int32_t* slot, const float* w,
                                 void* xs, const void* y, float* dw, mtk_stream stream) {
    if (const int rc = rows_check("mtk_rows_dispatch", n_rows, k, D, x_ld, dtype)) return rc;
    if (n_rows == 0) return MTK_OK;
    if (!x || !slot || (!xs && !dw) || ((y != nullptr) != (dw != nullptr))) MTK_FAIL(MTK_ERR_ARG, "mtk_rows_dispatch: null pointer");
    mtk_by_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        const int64_t touched = n_rows * D * (int64_t)sizeof(T) * (1 + k + (y ? k : 0));
        RowsArgs a{n_rows, n_rows * k, D, x_ld, k, slot, w, lanes_per_row(D, mtk_piece<T>::n), touched > kCaches};
        const unsigned grid = rows_grid(a);
        const T* xp = (const T*)x;
        const hipStream_t s = (hipStream_t)stream;
        by_flags(w != nullptr, dw != nullptr, k, [&](auto tw, auto td, auto tk) {
            k_dispatch<T, decltype(tw)::value, decltype(td)::value, decltype(tk)::value><<<grid, 256, 0, s>>>(a, xp, (T*)xs, (const T*)y, dw);
        });
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
        RowsArgs a{n_rows, n_rows * k, D, y_ld, k, slot, w, lanes_per_row(D, mtk_piece<T>::n), n_rows * D * (int64_t)sizeof(T) * (1 + k) > kCaches};
        const unsigned grid = rows_grid(a);
        const hipStream_t s = (hipStream_t)stream;
        by_flags(w != nullptr, false, k, [&](auto tw, auto, auto tk) { k_combine<T, decltype(tw)::value, decltype(tk)::value><<<grid, 256, 0, s>>>(a, (const T*)y, (T*)out); });
    });
    MTK_HIP(hipGetLastError());
    return MTK_OK;
}
