// mtk_adapter.hip — a linear layer shared by many models with one low-rank update per model, on rows sorted by model.
//
//   y = act(x W^T + b + s_e (x A_e^T) B_e^T)            rows offsets[e] .. offsets[e + 1] - 1 belong to model e,
//   dx = g W + s_e (g B_e) A_e                          rows from offsets[E] on have the shared layer alone
//   dA_e = s_e (g B_e)^T x,   dB_e = g^T (s_e x A_e^T)  g = dy, masked by y > 0 under a ReLU
//
// The shared product is a dense GEMM over all rows whatever model they belong to; what is per model is thin.  So:
//   k_shrink   u = s_e x A_e^T (M x r), 32 rows a workgroup, the reduction over the layer's width split over its waves;
//   k_linear   the dense tile, whose epilogue adds u B_e^T: a tile walks the models that own its rows (one, for most tiles), the
//              few extra MFMAs take u and B_e straight from memory;
//   k_wgrad    the factors' gradients over chunks of rows, joined in a fixed order by k_wgrad_join (no atomics).
// The backward of x is the same two kernels on g with W, A_e, B_e transposed first (W is small beside the rows).
// A row's product never meets another model's factors in an accumulator (0 x inf is NaN): products are made per model and
// SELECTED by row, so one diverged model leaves the others' rows alone.
// u and t = s_e g B_e are rounded to the rows' type (they are MFMA operands); every sum is in fp32.
#include "mtk_lowp.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef mtk_bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef mtk_f16 f16x8 __attribute__((ext_vector_type(8)));

// MFMA over one 16-byte piece per lane: k = 16 (32 x 32 tiles) or 32 (16 x 16) for 16-bit types.  fp32 takes the piece's four values in
// four instructions; which k a lane half holds does not matter as long as both operands agree, so the pieces are the same.
__device__ __forceinline__ f32x16 mma32(const mtk_vec<mtk_bf16>& a, const mtk_vec<mtk_bf16>& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(const mtk_vec<mtk_f16>& a, const mtk_vec<mtk_f16>& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(const mtk_vec<float>& a, const mtk_vec<float>& b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f32x4 mma16(const mtk_vec<mtk_bf16>& a, const mtk_vec<mtk_bf16>& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(const mtk_vec<mtk_f16>& a, const mtk_vec<mtk_f16>& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <typename T> __device__ __forceinline__ mtk_vec<T> zero_piece() {
    mtk_vec<T> v;
#pragma unroll
    for (int i = 0; i < mtk_piece<T>::n; ++i) v.v[i] = T(0);
    return v;
}

// elements of the low rank as stored in u: whole MFMA steps
template <typename T> constexpr int kRankStep = 32 / (int)sizeof(T);
template <typename T> __host__ __device__ constexpr int rank_pad(int r) { return (r + kRankStep<T> - 1) / kRankStep<T> * kRankStep<T>; }
inline int rank_pad_of(int r, int dtype) { return dtype == MTK_DT_F32 ? rank_pad<float>(r) : rank_pad<mtk_bf16>(r); }
constexpr int kRankT = 16;  // rows of u^T come in whole 16s

// The models that own rows [at, end): each call yields one (e, first row, behind its last row).  Offsets are clamped and every step moves
// forward, so whatever they hold no row outside [at, end) is named and the walk ends.
struct Owners {
    const int32_t* off;
    int E;
    int64_t at, end;
    __device__ bool next(int& e, int64_t& a, int64_t& b) {
        while (at < end) {
            int lo = 0, hi = E + 1;  // number of offsets <= at
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (off[mid] <= at) lo = mid + 1;
                else hi = mid;
            }
            if (lo > E) return false;  // behind the last model's rows
            const int64_t to = off[lo] < end ? off[lo] : end;
            if (lo == 0) {
                at = to;
                continue;
            }
            e = lo - 1;
            a = at;
            b = to;
            at = to;
            return true;
        }
        return false;
    }
};

// ------------------------------------------------------------------------------------------------------------------ shrink
struct ShrinkArgs {
    int64_t M;
    int K, r, rp, E;
    int64_t x_ld;
    const int32_t* offsets;
    const float* scales;
    float scale;
    int64_t Mp;  // row stride of uT
};

// u[row][j] = s_e sum_k x[row][k] F_e[j][k] (F: [E][r][K]); with uT also its transpose, which the factors' gradients multiply
template <typename T, int NW>
__global__ __launch_bounds__(64 * NW) void k_shrink(ShrinkArgs g, const T* __restrict__ x, const T* __restrict__ F, T* __restrict__ u, T* __restrict__ uT) {
    constexpr int V = mtk_piece<T>::n, KB = 8 * V;  // a k-block is a 128-byte line of a row
    __shared__ float part[NW][32][33];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, hh = lane >> 5;
    const int64_t m0 = (int64_t)blockIdx.x * 32;
    const int64_t end = m0 + 32 < g.M ? m0 + 32 : g.M;
    const int64_t row = m0 + li < g.M ? m0 + li : g.M - 1;
    const T* xr = x + row * g.x_ld;
    const int jw = uT ? (int)mtk_up(g.rp, kRankT) : g.rp;
    for (int j0 = 0; j0 < jw; j0 += 32) {
        Owners own{g.offsets, g.E, m0, end};
        int e;
        int64_t a, b;
        float keep[32 * 32 / (64 * NW)];
#pragma unroll
        for (int i = 0; i < 32 * 32 / (64 * NW); ++i) keep[i] = 0.f;
        while (own.next(e, a, b)) {
            const int j = j0 + li < g.r ? j0 + li : g.r - 1;
            const T* fr = F + ((int64_t)e * g.r + j) * g.K;
            f32x16 acc = {};
            for (int k0 = wave * KB; k0 < g.K; k0 += NW * KB) {
                mtk_vec<T> xa[4], fa[4];
                if (k0 + KB <= g.K) {
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        const int k = k0 + (2 * s + hh) * V;
                        xa[s] = mtk_ld(xr + k);
                        fa[s] = mtk_ld(fr + k);
                    }
                } else {
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        const int k = k0 + (2 * s + hh) * V;
                        xa[s] = mtk_ld_n(xr + k, g.K - k);
                        fa[s] = mtk_ld_n(fr + k, g.K - k);
                    }
                }
#pragma unroll
                for (int s = 0; s < 4; ++s) acc = mma32(fa[s], xa[s], acc);
            }
            // D[j][record]: lane -> record, register -> j = (reg & 3) + 8 (reg >> 2) + 4 (lane >> 5)
#pragma unroll
            for (int q = 0; q < 16; ++q) part[wave][li][(q & 3) + 8 * (q >> 2) + 4 * hh] = acc[q];
            __syncthreads();
            const float s = g.scales ? g.scales[e] : g.scale;
#pragma unroll
            for (int i = 0; i < 32 * 32 / (64 * NW); ++i) {
                const int q = tid + i * 64 * NW, rr = q >> 5, jj = q & 31;
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < NW; ++w) v += part[w][rr][jj];
                if (m0 + rr >= a && m0 + rr < b && j0 + jj < g.r) keep[i] = s * v;
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 32 * 32 / (64 * NW); ++i) {
            const int q = tid + i * 64 * NW, rr = q >> 5, jj = q & 31;
            if (m0 + rr < g.M && j0 + jj < g.rp) u[(m0 + rr) * g.rp + j0 + jj] = (T)keep[i];
            if (uT) part[0][rr][jj] = keep[i];
        }
        if (uT) {  // through LDS: a thread per (j, record), records fastest
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 32 * 32 / (64 * NW); ++i) {
                const int q = tid + i * 64 * NW, rr = q & 31, jj = q >> 5;
                if (j0 + jj < jw) uT[(int64_t)(j0 + jj) * g.Mp + m0 + rr] = (T)part[0][rr][jj];  // Mp covers whole tiles of 32 rows
            }
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------ linear
struct LinearArgs {
    int64_t M, x_ld;
    int N, K, r, rp, E;
    const int32_t* offsets;
    int relu;
};

constexpr int TM = 128, TN = 128;

// y = act(x W^T + b + u B_e^T): tiles of 128 rows x 128 features, four waves of 64 x 64, k-blocks of 128 bytes double buffered in LDS.
// Weights are the MFMA's A operand: a lane then holds consecutive features of one record, which leave as 8- or 16-byte pieces.
template <typename T>
__global__ __launch_bounds__(256) void k_linear(LinearArgs g, const T* __restrict__ x, const T* __restrict__ W, const T* __restrict__ bias, const T* __restrict__ u,
                                                const T* __restrict__ up, T* __restrict__ y) {
    constexpr int V = mtk_piece<T>::n, KB = 8 * V;
    __shared__ __attribute__((aligned(16))) unsigned char lds[2][2][TM * 128];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, hh = lane >> 5;
    const int wr = wave >> 1, wc = wave & 1;
    const int nb = (g.N + TN - 1) / TN;
    const int64_t m0 = (int64_t)(blockIdx.x / nb) * TM;
    const int n0 = (int)(blockIdx.x % nb) * TN;

    mtk_vec<T> px[4], pw[4];
    auto fetch = [&](int k0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = tid + i * 256, rr = p >> 3, k = k0 + (p & 7) * V;
            const int64_t row = m0 + rr < g.M ? m0 + rr : g.M - 1;
            const int n = n0 + rr < g.N ? n0 + rr : g.N - 1;
            const T *xp = x + row * g.x_ld + k, *wp = W + (int64_t)n * g.K + k;
            if (k0 + KB <= g.K) {
                px[i] = mtk_ld(xp);
                pw[i] = mtk_ld(wp);
            } else {
                px[i] = mtk_ld_n(xp, g.K - k);
                pw[i] = mtk_ld_n(wp, g.K - k);
            }
        }
    };
    // piece p of row r sits at slot p ^ ((r >> 1) & 7): the 16 lanes that ds_read_b128 serves together then touch 16 different slots
    auto put = [&](int buf) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = tid + i * 256, rr = p >> 3, at = rr * 128 + (((p & 7) ^ ((rr >> 1) & 7)) * 16);
            *reinterpret_cast<uint4*>(&lds[buf][0][at]) = __builtin_bit_cast(uint4, px[i]);
            *reinterpret_cast<uint4*>(&lds[buf][1][at]) = __builtin_bit_cast(uint4, pw[i]);
        }
    };
    auto frag = [&](int buf, int op, int rr, int kp) {
        return __builtin_bit_cast(mtk_vec<T>, *reinterpret_cast<const uint4*>(&lds[buf][op][rr * 128 + ((kp ^ ((rr >> 1) & 7)) * 16)]));
    };

    f32x16 acc[2][2] = {};
    const int nkb = (g.K + KB - 1) / KB;
    fetch(0);
    put(0);
    __syncthreads();
    for (int kb = 0; kb < nkb; ++kb) {
        if (kb + 1 < nkb) fetch((kb + 1) * KB);
        const int buf = kb & 1;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            mtk_vec<T> fx[2], fw[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                fx[q] = frag(buf, 0, wr * 64 + q * 32 + li, 2 * s + hh);
                fw[q] = frag(buf, 1, wc * 64 + q * 32 + li, 2 * s + hh);
            }
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) acc[mt][nt] = mma32(fw[nt], fx[mt], acc[mt][nt]);
        }
        if (kb + 1 < nkb) put(buf ^ 1);
        __syncthreads();
    }

    int64_t rows[2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) rows[mt] = m0 + wr * 64 + mt * 32 + li;
    if (up) {
        const int64_t w0 = m0 + wr * 64;
        Owners own{g.offsets, g.E, w0, w0 + 64 < g.M ? w0 + 64 : g.M};
        int e;
        int64_t a, b;
        while (own.next(e, a, b)) {
            f32x16 low[2][2] = {};
            for (int j = hh * V; j < g.rp; j += 2 * V) {
                mtk_vec<T> fu[2], fb[2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int64_t row = rows[q] < g.M ? rows[q] : g.M - 1;
                    const int n = n0 + wc * 64 + q * 32 + li, nc = n < g.N ? n : g.N - 1;
                    const T* bp = up + ((int64_t)e * g.N + nc) * g.r + j;
                    fu[q] = mtk_ld(u + row * g.rp + j);
                    fb[q] = j + V <= g.r ? mtk_ld(bp) : mtk_ld_n(bp, g.r - j);
                }
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt) low[mt][nt] = mma32(fb[nt], fu[mt], low[mt][nt]);
            }
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                const bool mine = rows[mt] >= a && rows[mt] < b;
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int q = 0; q < 16; ++q) acc[mt][nt][q] += mine ? low[mt][nt][q] : 0.f;
            }
        }
    }
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int n = n0 + wc * 64 + nt * 32 + 8 * q + 4 * hh;
            float bv[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) bv[j] = bias && n + j < g.N ? (float)bias[n + j] : 0.f;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                if (rows[mt] >= g.M) continue;
                T* yp = y + rows[mt] * g.N + n;
                struct __attribute__((packed, aligned(alignof(T)), may_alias)) Quad { T v[4]; } o;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float v = acc[mt][nt][4 * q + j] + bv[j];
                    if (g.relu) v = v < 0.f ? 0.f : v;  // NaN stays
                    o.v[j] = (T)v;
                }
                if (n + 4 <= g.N) *reinterpret_cast<Quad*>(yp) = o;
                else
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (n + j < g.N) yp[j] = o.v[j];
            }
        }
}

// ------------------------------------------------------------------------------------------------- the factors' gradients
struct WgradArgs {
    int64_t M, x_ld, Mp;
    int D, r, rp, E;
    int chunk;   // rows of a workgroup's chunk, a multiple of 32
    const int32_t* offsets;
};

// part[c + e][j][d] = sum over the rows of chunk c that model e owns of u[row][j] x[row][d].  Walking the chunks, each step to the next
// (chunk, model) pair raises c, e or both, so c + e numbers the pairs without a gap's worth of bookkeeping.
// 16-bit types: MFMA 16 x 16 x 32, the rows are its k.  u^T gives a lane's eight rows of one j as one piece; x's eight rows of eight
// columns come as eight pieces and are turned in registers.  Rows of other models are zeroed in BOTH operands (0 x inf).
template <typename T, int JT>
__global__ __launch_bounds__(256) void k_wgrad16(WgradArgs g, int j0, const T* __restrict__ uT, const T* __restrict__ x, float* __restrict__ part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, q = lane >> 4;
    const int c0 = (blockIdx.x * 4 + wave) * 128 + li * 8;
    if ((blockIdx.x * 4 + wave) * 128 >= g.D) return;
    const int cols = g.D - c0;
    const int64_t lo = (int64_t)blockIdx.y * g.chunk, hi = lo + g.chunk < g.M ? lo + g.chunk : g.M;
    Owners own{g.offsets, g.E, lo, hi};
    int e;
    int64_t a, b;
    const int jp = (int)mtk_up(g.r, kRankT);
    while (own.next(e, a, b)) {
        f32x4 acc[JT][8] = {};
        for (int64_t r0 = a / 32 * 32; r0 < b; r0 += 32) {
            const int64_t rr = r0 + q * 8;
            mtk_vec<T> xv[8], ut[JT];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int64_t row = rr + i;
                const bool in = row >= a && row < b;
                const T* xp = x + row * g.x_ld + c0;
                xv[i] = in && cols >= 8 ? mtk_ld(xp) : mtk_ld_n(xp, in ? cols : 0);
            }
#pragma unroll
            for (int t = 0; t < JT; ++t) {
                ut[t] = mtk_ld(uT + (int64_t)(j0 + t * 16 + li) * g.Mp + rr);
#pragma unroll
                for (int i = 0; i < 8; ++i) ut[t].v[i] = rr + i >= a && rr + i < b ? ut[t].v[i] : T(0);
            }
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                mtk_vec<T> col;
#pragma unroll
                for (int i = 0; i < 8; ++i) col.v[i] = xv[i].v[c];
#pragma unroll
                for (int t = 0; t < JT; ++t) acc[t][c] = mma16(ut[t], col, acc[t][c]);
            }
        }
        // D[j][column lane]: register -> j = 4 (lane >> 4) + reg, column li of the c-th set is c0 + c
        float* o = part + (int64_t)(blockIdx.y + e) * jp * g.D;
#pragma unroll
        for (int t = 0; t < JT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = j0 + t * 16 + q * 4 + i;
                float* op = o + (int64_t)j * g.D + c0;
                mtk_vec<float> v0, v1;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    v0.v[c] = acc[t][c][i];
                    v1.v[c] = acc[t][c + 4][i];
                }
                if (j >= g.r) continue;
                if (cols >= 8) {
                    mtk_st(op, v0);
                    mtk_st(op + 4, v1);
                } else if (cols > 0) {
                    mtk_st_n(op, v0, cols);
                    mtk_st_n(op + 4, v1, cols - 4);
                }
            }
    }
}

// fp32: MFMA 16 x 16 x 4, a lane holds one row's four columns and one j; nothing to turn
template <int JT>
__global__ __launch_bounds__(256) void k_wgrad32(WgradArgs g, int j0, const float* __restrict__ u, const float* __restrict__ x, float* __restrict__ part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, q = lane >> 4;
    const int c0 = (blockIdx.x * 4 + wave) * 64 + li * 4;
    if ((blockIdx.x * 4 + wave) * 64 >= g.D) return;
    const int cols = g.D - c0;
    const int64_t lo = (int64_t)blockIdx.y * g.chunk, hi = lo + g.chunk < g.M ? lo + g.chunk : g.M;
    Owners own{g.offsets, g.E, lo, hi};
    int e;
    int64_t a, b;
    const int jp = (int)mtk_up(g.r, kRankT);
    while (own.next(e, a, b)) {
        f32x4 acc[JT][4] = {};
        for (int64_t r0 = a / 16 * 16; r0 < b; r0 += 16) {
            mtk_vec<float> xv[4];
            float ut[4][JT];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int64_t row = r0 + s * 4 + q;
                const bool in = row >= a && row < b;
                const float* xp = x + row * g.x_ld + c0;
                xv[s] = in && cols >= 4 ? mtk_ld(xp) : mtk_ld_n(xp, in ? cols : 0);
#pragma unroll
                for (int t = 0; t < JT; ++t) {
                    const int j = j0 + t * 16 + li;
                    ut[s][t] = in && j < g.rp ? u[row * g.rp + j] : 0.f;
                }
            }
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int t = 0; t < JT; ++t)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[t][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(ut[s][t], xv[s].v[c], acc[t][c], 0, 0, 0);
        }
        float* o = part + (int64_t)(blockIdx.y + e) * jp * g.D;
#pragma unroll
        for (int t = 0; t < JT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = j0 + t * 16 + q * 4 + i;
                if (j >= g.r) continue;
                mtk_vec<float> v;
#pragma unroll
                for (int c = 0; c < 4; ++c) v.v[c] = acc[t][c][i];
                if (cols >= 4) mtk_st(o + (int64_t)j * g.D + c0, v);
                else if (cols > 0) mtk_st_n(o + (int64_t)j * g.D + c0, v, cols);
            }
    }
}

// out[e] = sum of model e's chunks in ascending order; [r][D], or [D][r] when `turn`.  A model without rows gets zeros.
template <typename T>
__global__ __launch_bounds__(256) void k_wgrad_join(WgradArgs g, int turn, const float* __restrict__ part, T* __restrict__ out) {
    const int e = blockIdx.y;
    const int jp = (int)mtk_up(g.r, kRankT);
    const int64_t n = (int64_t)g.r * g.D;
    int64_t a = g.offsets[e], b = g.offsets[e + 1];
    a = a < 0 ? 0 : a;
    b = b < g.M ? b : g.M;
    const int64_t ca = a / g.chunk, cb = b > a ? (b - 1) / g.chunk : ca - 1;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t j = i / g.D, d = i - j * g.D;
        float s = 0.f;
        for (int64_t c = ca; c <= cb; ++c) s += part[((c + e) * jp + j) * g.D + d];
        out[(int64_t)e * n + (turn ? d * g.r + j : i)] = (T)s;
    }
}

// ------------------------------------------------------------------------------------------------------------------ helpers
// [batch][R][C] -> [batch][C][R]
template <typename T>
__global__ __launch_bounds__(256) void k_turn(const T* __restrict__ in, T* __restrict__ out, int R, int C) {
    __shared__ T tile[32][33];
    const int64_t base = (int64_t)blockIdx.z * R * C;
    const int c0 = blockIdx.x * 32, r0 = blockIdx.y * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    for (int i = ty; i < 32; i += 8)
        if (r0 + i < R && c0 + tx < C) tile[i][tx] = in[base + (int64_t)(r0 + i) * C + c0 + tx];
    __syncthreads();
    for (int i = ty; i < 32; i += 8)
        if (c0 + i < C && r0 + tx < R) out[base + (int64_t)(c0 + i) * R + r0 + tx] = tile[tx][i];
}

// g = dy, 0 where y <= 0
template <typename T>
__global__ __launch_bounds__(256) void k_relu_grad(int64_t n, const T* __restrict__ y, const T* __restrict__ dy, T* __restrict__ gz) {
    constexpr int V = mtk_piece<T>::n;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V; i < n; i += (int64_t)gridDim.x * 256 * V) {
        const int left = n - i < V ? (int)(n - i) : V;
        const mtk_vec<T> a = left == V ? mtk_ld(y + i) : mtk_ld_n(y + i, left);
        mtk_vec<T> d = left == V ? mtk_ld(dy + i) : mtk_ld_n(dy + i, left);
#pragma unroll
        for (int k = 0; k < V; ++k) d.v[k] = (float)a.v[k] <= 0.f ? T(0) : d.v[k];
        if (left == V) mtk_st(gz + i, d);
        else mtk_st_n(gz + i, d, left);
    }
}

int wgrad_chunk(int64_t M, int D) {
    const int64_t want = M * ((D + 127) / 128) / 2048;  // about 2048 waves
    const int64_t c = mtk_up(want < 1 ? 1 : want, 32);
    return (int)(c < 64 ? 64 : (c > 1024 ? 1024 : c));
}
int64_t wgrad_part(int64_t M, int D, int r, int E) {
    return ((M + wgrad_chunk(M, D) - 1) / wgrad_chunk(M, D) + E) * mtk_up(r, kRankT) * D;
}

template <typename T>
void shrink(const ShrinkArgs& g, const T* x, const T* F, T* u, T* uT, hipStream_t s) {
    k_shrink<T, 4><<<(unsigned)((g.M + 31) / 32), 256, 0, s>>>(g, x, F, u, uT);
}
template <typename T>
void linear(const LinearArgs& g, const T* x, const T* W, const T* bias, const T* u, const T* up, T* y, hipStream_t s) {
    const unsigned grid = (unsigned)((g.M + TM - 1) / TM * ((g.N + TN - 1) / TN));
    k_linear<T><<<grid, 256, 0, s>>>(g, x, W, bias, u, up, y);
}
template <typename T, int JT>
void wgrad_launch(const WgradArgs& g, int j0, const T* u, const T* uT, const T* x, float* part, hipStream_t s) {
    const unsigned nch = (unsigned)((g.M + g.chunk - 1) / g.chunk);
    if constexpr (sizeof(T) == 4) k_wgrad32<JT><<<dim3((g.D + 255) / 256, nch), 256, 0, s>>>(g, j0, u, x, part);
    else k_wgrad16<T, JT><<<dim3((g.D + 511) / 512, nch), 256, 0, s>>>(g, j0, uT, x, part);
}
template <typename T>
void wgrad(const WgradArgs& g, int turn, const T* u, const T* uT, const T* x, float* part, T* out, hipStream_t s) {
    for (int j0 = 0; j0 < g.r; j0 += 64) {
        if (g.r - j0 > 32) wgrad_launch<T, 4>(g, j0, u, uT, x, part, s);
        else if (g.r - j0 > 16) wgrad_launch<T, 2>(g, j0, u, uT, x, part, s);
        else wgrad_launch<T, 1>(g, j0, u, uT, x, part, s);
    }
    const int64_t n = (int64_t)g.r * g.D;
    const unsigned nx = (unsigned)((n + 255) / 256 < 1024 ? (n + 255) / 256 : 1024);
    k_wgrad_join<T><<<dim3(nx, g.E), 256, 0, s>>>(g, turn, part, out);
}
template <typename T>
void turn(const T* in, T* out, int R, int C, int batch, hipStream_t s) {
    k_turn<T><<<dim3((C + 31) / 32, (R + 31) / 32, batch), 256, 0, s>>>(in, out, R, C);
}

// where the parts of a buffer lie, in bytes, each on 256
struct Layout {
    int64_t at = 0;
    int64_t take(int64_t bytes) {
        const int64_t a = at;
        at += mtk_up(bytes, 256);
        return a;
    }
};
struct Saved {
    int64_t u, uT, bytes, Mp;
    Saved(int64_t M, int r, int dtype) {
        Layout l;
        Mp = mtk_up(M, 32);
        u = l.take(M * rank_pad_of(r, dtype) * mtk_dtype_size(dtype));
        uT = dtype == MTK_DT_F32 ? l.at : l.take(Mp * mtk_up(r, 64) * mtk_dtype_size(dtype));
        bytes = l.at;
    }
};
struct Work {
    int64_t Wt, At, Bt, t, g, part, bytes;
    Work(int64_t M, int din, int dout, int r, int E, int dtype, bool relu) {
        const int64_t z = mtk_dtype_size(dtype);
        Layout l;
        Wt = l.take((int64_t)din * dout * z);
        At = l.take((int64_t)E * r * din * z);
        Bt = l.take((int64_t)E * r * dout * z);
        t = l.take(Saved(M, r, dtype).bytes);
        g = l.take(relu ? M * dout * z : 0);
        const int64_t pa = wgrad_part(M, din, r, E), pb = wgrad_part(M, dout, r, E);
        part = l.take((pa > pb ? pa : pb) * 4);
        bytes = l.at;
    }
};

int adapter_check(const char* who, int64_t M, int din, int dout, int r, int E, int dtype, int64_t x_ld, int act) {
    if (M < 0 || din < 1 || dout < 1 || r < 1 || E < 1 || x_ld < 0) MTK_FAIL(MTK_ERR_ARG, "%s: bad sizes (rows %lld, %d -> %d, rank %d, %d models)", who, (long long)M, din, dout, r, E);
    if (!mtk_dtype_ok(dtype)) MTK_FAIL(MTK_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
    if (act != 0 && act != 1) MTK_FAIL(MTK_ERR_UNSUPPORTED, "%s: activation %d", who, act);
    if (r > MTK_ADAPTER_MAX_RANK) MTK_FAIL(MTK_ERR_UNSUPPORTED, "%s: rank %d exceeds %d", who, r, MTK_ADAPTER_MAX_RANK);
    if (E > MTK_ROUTE_MAX_GROUPS) MTK_FAIL(MTK_ERR_UNSUPPORTED, "%s: %d models exceed %d", who, E, MTK_ROUTE_MAX_GROUPS);
    if (din > MTK_ADAPTER_MAX_WIDTH || dout > MTK_ADAPTER_MAX_WIDTH) MTK_FAIL(MTK_ERR_UNSUPPORTED, "%s: %d -> %d features (up to %d)", who, din, dout, MTK_ADAPTER_MAX_WIDTH);
    if (M > MTK_ADAPTER_MAX_ROWS) MTK_FAIL(MTK_ERR_UNSUPPORTED, "%s: %lld rows exceed %lld", who, (long long)M, (long long)MTK_ADAPTER_MAX_ROWS);
    return MTK_OK;
}

}  // namespace

extern "C" int64_t mtk_adapter_saved_bytes(int64_t M, int r, int dtype) {
    return M > 0 && r > 0 && mtk_dtype_ok(dtype) ? Saved(M, r, dtype).bytes : 0;
}
extern "C" int64_t mtk_adapter_work_bytes(int64_t M, int din, int dout, int r, int E, int dtype, int act) {
    return M > 0 && din > 0 && dout > 0 && r > 0 && E > 0 && mtk_dtype_ok(dtype) ? Work(M, din, dout, r, E, dtype, act == 1).bytes : 0;
}

extern "C" int mtk_adapter_forward(int64_t M, int din, int dout, int r, int E, int dtype, const void* x, int64_t x_ld, const void* W, const void* bias,
                                   const void* down, const void* up, const int32_t* offsets, const float* scales, double scale, int act, int keep,
                                   void* y, void* saved, int64_t saved_bytes, mtk_stream stream) {
    if (const int rc = adapter_check("mtk_adapter_forward", M, din, dout, r, E, dtype, x_ld, act)) return rc;
    if (M == 0) return MTK_OK;
    if (!x || !W || !down || !up || !offsets || !y || !saved) MTK_FAIL(MTK_ERR_ARG, "mtk_adapter_forward: null pointer");
    const Saved sv(M, r, dtype);
    if (saved_bytes < sv.bytes) MTK_FAIL(MTK_ERR_ARG, "mtk_adapter_forward: a buffer of %lld bytes for the low-rank rows, %lld needed", (long long)saved_bytes, (long long)sv.bytes);
    mtk_by_type(dtype, [&](auto tag) {
        typedef decltype(tag) T;
        const hipStream_t s = (hipStream_t)stream;
        T* u = (T*)((char*)saved + sv.u);
        T* uT = keep && sizeof(T) == 2 ? (T*)((char*)saved + sv.uT) : nullptr;
        shrink<T>(ShrinkArgs{M, din, r, rank_pad<T>(r), E, x_ld, offsets, scales, (float)scale, sv.Mp}, (const T*)x, (const T*)down, u, uT, s);
        linear<T>(LinearArgs{M, x_ld, dout, din, r, rank_pad<T>(r), E, offsets, act}, (const T*)x, (const T*)W, (const T*)bias, u, (const T*)up, (T*)y, s);
    });
    MTK_HIP(hipGetLastError());
    return MTK_OK;
}

extern "C" int mtk_adapter_backward(int64_t M, int din, int dout, int r, int E, int dtype, const void* x, int64_t x_ld, const void* W, const void* down,
                                    const void* up, const int32_t* offsets, const float* scales, double scale, int act, const void* y, const void* dy,
                                    const void* saved, void* dx, void* ddown, void* dup, void* work, int64_t work_bytes, mtk_stream stream) {
    if (const int rc = adapter_check("mtk_adapter_backward", M, din, dout, r, E, dtype, x_ld, act)) return rc;
    if (M == 0) return MTK_OK;
    if (!x || !W || !down || !up || !offsets || !dy || !saved || !work || (act && !y)) MTK_FAIL(MTK_ERR_ARG, "mtk_adapter_backward: null pointer");
    const Saved sv(M, r, dtype);
    const Work wk(M, din, dout, r, E, dtype, act == 1);
    if (work_bytes < wk.bytes) MTK_FAIL(MTK_ERR_ARG, "mtk_adapter_backward: workspace of %lld bytes, %lld needed", (long long)work_bytes, (long long)wk.bytes);
    mtk_by_type(dtype, [&](auto tag) {
        typedef decltype(tag) T;
        const hipStream_t s = (hipStream_t)stream;
        char* wb = (char*)work;
        const int rp = rank_pad<T>(r);
        const T *u = (const T*)((const char*)saved + sv.u), *uT = (const T*)((const char*)saved + sv.uT);
        T *t = (T*)(wb + wk.t + sv.u), *tT = (T*)(wb + wk.t + sv.uT);
        const T* g = (const T*)dy;
        if (act) {
            T* gz = (T*)(wb + wk.g);
            const int64_t n = M * dout, nb = (n + 256 * mtk_piece<T>::n - 1) / (256 * mtk_piece<T>::n);
            k_relu_grad<T><<<(unsigned)(nb < 65536 ? nb : 65536), 256, 0, s>>>(n, (const T*)y, g, gz);
            g = gz;
        }
        if (dx || ddown) {
            T* Bt = (T*)(wb + wk.Bt);
            turn<T>((const T*)up, Bt, dout, r, E, s);
            shrink<T>(ShrinkArgs{M, dout, r, rp, E, dout, offsets, scales, (float)scale, sv.Mp}, g, Bt, t, ddown && sizeof(T) == 2 ? tT : nullptr, s);
        }
        if (dx) {
            T *Wt = (T*)(wb + wk.Wt), *At = (T*)(wb + wk.At);
            turn<T>((const T*)W, Wt, dout, din, 1, s);
            turn<T>((const T*)down, At, r, din, E, s);
            linear<T>(LinearArgs{M, dout, din, dout, r, rp, E, offsets, 0}, g, Wt, nullptr, t, At, (T*)dx, s);
        }
        float* part = (float*)(wb + wk.part);
        if (ddown) wgrad<T>(WgradArgs{M, x_ld, sv.Mp, din, r, rp, E, wgrad_chunk(M, din), offsets}, 0, t, tT, (const T*)x, part, (T*)ddown, s);
        if (dup) wgrad<T>(WgradArgs{M, dout, sv.Mp, dout, r, rp, E, wgrad_chunk(M, dout), offsets}, 1, u, uT, g, part, (T*)dup, s);
    });
    MTK_HIP(hipGetLastError());
    return MTK_OK;
}
