// mtk_adapter.hip — a linear layer shared by many models with one low-rank update per model, on rows sorted by model.
//
//   y = act(x W^T + b + s_e (x A_e^T) B_e^T)            rows offsets[e] .. offsets[e + 1] - 1 belong to model e,
//   dx = g W + s_e (g B_e) A_e                          rows from offsets[E] on have the shared layer alone
//   dA_e = s_e (g B_e)^T x,   dB_e = g^T (s_e x A_e^T)  g = dy, masked by y > 0 under a ReLU
//
// The shared product is a dense GEMM over all rows whatever model they belong to; what is per model is thin.  So:
//   k_shrink   u = s_e x A_e^T (M x r), bound by reading x; what has to be laid out for the products rides in its launch (k_prep alone only
//              where the shrink itself needs it);
//   k_linear   the dense tiles, with u B_e^T as their last k-blocks; k_linear_few for few rows;
//   k_wgrad    the factors' gradients over chunks of rows, joined in a fixed order by k_wgrad_join (no atomics).
// The backward of x is the same two kernels on g with W, A_e, B_e transposed first (W is small beside the rows).
// One diverged model leaves the others' rows alone, to the bit: what is not finite never meets another model's rows in an accumulator
// (0 x inf is NaN), their products are made per model and SELECTED by row.
// Every sum is in fp32.  u and t = s_e g B_e are MFMA operands, so with 16-bit rows they are 16-bit numbers, and more than one each: a single rounded
// number would add as much error as the result's own rounding, and all of a row's at once.  A row of u holds them in sections side by side:
//   bf16  two, u = hi + lo (2^-18 of u), against B_e twice; for ranks up to 32 the line of 64 numbers holds both
//   fp16  three bf16 numbers, u = h + m + l (2^-27), against B_e = b + c, two bf16 numbers (exact): h b + m b + l b + h c + m c.  Not fp16 numbers:
//         t is small (the factors start at zero, gradients are small), and below 2^-14 fp16 has fewer bits with every binade, 6e-8 of
//         absolute error; at the other end u passes 65,504 where y does not.  bf16 has fp32's exponents.  One line up to rank 12.
#include <type_traits>

#include "mtk_low_piece.h"
#include "mtk_lowp.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
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

__device__ __forceinline__ f32x4 mma16(const mtk_vec<float>& a, const mtk_vec<float>& b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
}

// A k-block is one 128-byte line of a row.  A row of u is rank_pad elements, whole lines: kSections sections of `section` values, zeros behind the rank
// and behind the last.
template <typename T> constexpr int kLine = 128 / (int)sizeof(T);
template <typename T> constexpr bool kF16 = std::is_same<T, mtk_f16>::value;
template <typename T> using Low = typename std::conditional<kF16<T>, mtk_bf16, T>::type;  // what u is made of
template <typename T> constexpr int kParts = sizeof(T) == 4 ? 1 : kF16<T> ? 3 : 2;        // numbers of a value of u
template <typename T> constexpr int kSections = kF16<T> ? 5 : kParts<T>;
template <typename T> __host__ __device__ constexpr int section(int r) { return kF16<T> ? (r + 3) / 4 * 4 : (r + 31) / 32 * 32; }
constexpr int section_part(int s) { return s < 3 ? s : s - 3; }  // the number that section s holds
constexpr bool section_second(int s) { return s >= 3; }          // whether it meets the second number of B_e
// eight fp16 values as two bf16 numbers each, exactly (an infinity: inf and NaN)
__device__ __forceinline__ void two_numbers(const mtk_vec<mtk_f16>& v, mtk_vec<mtk_bf16>& b, mtk_vec<mtk_bf16>& c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float f = (float)v.v[i];
        b.v[i] = (mtk_bf16)f;
        c.v[i] = (mtk_bf16)(f - (float)b.v[i]);
    }
}
// the first of them, or the second
__device__ __forceinline__ mtk_vec<mtk_bf16> number_of(const mtk_vec<mtk_f16>& v, bool second) {
    mtk_vec<mtk_bf16> o;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float f = (float)v.v[i];
        o.v[i] = (mtk_bf16)(f - (second ? (float)(mtk_bf16)f : 0.f));
    }
    return o;
}
inline int rank_pad(int r, int dtype) {
    return dtype == MTK_DT_F32 ? section<float>(r) : dtype == MTK_DT_BF16 ? 2 * section<mtk_bf16>(r) : (int)mtk_up(5 * section<mtk_f16>(r), kLine<mtk_f16>);
}
// the numbers of v, largest first; what follows an infinity is 0
template <typename L, int N> __device__ __forceinline__ void parts_of(float v, L (&p)[N]) {
    p[0] = (L)v;
    if constexpr (N > 1) {
        float rest = fabsf((float)p[0]) <= 3.0e38f ? v - (float)p[0] : 0.f;
#pragma unroll
        for (int i = 1; i < N; ++i) {
            p[i] = (L)rest;
            rest -= (float)p[i];
        }
    }
}
constexpr int kRankT = 16;  // rows of u^T come in whole 16s

// The models that own rows [at, end): each call yields one (e, first row, behind its last row).  Whatever the offsets hold, every step moves
// forward and stays inside [at, end), so no other row is named and the walk ends.
// A wave's walk: its lanes hold an offset each, so a step is a ballot and not a chain of loads (beyond 64 offsets, one load a 64).
struct Owners {
    const int32_t* off;
    int E;
    int64_t at, end;
    int held;  // lane's offset of the first 64
    __device__ Owners(const int32_t* off_, int E_, int64_t at_, int64_t end_) : off(off_), E(E_), at(at_), end(end_) {
        const int lane = __lane_id();
        held = lane <= E ? off[lane] : 0x7fffffff;
    }
    __device__ int behind(int64_t row) const {  // offsets <= row
        int lo = __popcll(__ballot(held <= row));
        for (int i = 64; i <= E && lo == i; i += 64) {
            const int k = i + (int)__lane_id();
            lo += __popcll(__ballot((k <= E ? off[k] : 0x7fffffff) <= row));
        }
        return lo;
    }
    __device__ bool next(int& e, int64_t& a, int64_t& b) {
        while (at < end) {
            const int lo = behind(at);
            if (lo > E) return false;  // behind the last model's rows
            int64_t to = lo < 64 ? __builtin_amdgcn_readlane(held, lo) : __builtin_amdgcn_readfirstlane(off[lo]);
            to = to > at ? to : at + 1;
            to = to < end ? to : end;
            a = at;
            b = to;
            at = to;
            if (lo == 0) continue;
            e = lo - 1;
            return true;
        }
        return false;
    }
};

// The models of a row tile: the first, how many (0: none, or too many for a run of k-blocks each), whether some rows are not the first's, whether
// there are too many.
constexpr int kTileModels = 8;
struct TileModels {
    int e, count, ranged, many;
    __device__ int packed() const { return e | count << 16 | ranged << 24 | many << 25; }
    __device__ static TileModels of(int packed) { return TileModels{packed & 0xffff, packed >> 16 & 0xff, packed >> 24 & 1, packed >> 25 & 1}; }
    // Of rows first .. first + rows - 1 of M.  Whatever the offsets hold, the models named are below E, and all who ask get the same.
    __device__ static TileModels of_tile(const Owners& own, int64_t first, int rows, int64_t M, int E) {
        const int64_t last = (first + rows < M ? first + rows : M) - 1;
        const int e0 = own.behind(first) - 1, e1 = own.behind(last) - 1;  // -1: before the first offset, E: behind the last (no model)
        TileModels m = {e0 < 0 ? 0 : e0, 0, e0 != e1, 0};
        m.count = (e1 < E ? e1 : E - 1) - m.e + 1;
        if (m.count < 0) m.count = 0;
        if (m.count > kTileModels) m.count = 0, m.many = 1;
        if (m.count == 0) m.e = m.ranged = 0;
        return m;
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
    void* pairs;  // with BM > 0: the rows of tiles that models share, once a model (see k_linear)
    int BM;
    int turns, tiles;  // workgroups: turns x tiles
};

// u[row][j] = s_e sum_k x[row][k] F_e[j][k] (F: [E][r][K]); with uT also its transpose, which the factors' gradients multiply.
// Bound by reading x.  16 x 16 MFMA tiles: RR sets of 16 rows against RT tiles of 16 j, so a rank of 16 wastes nothing; a wave streams its rows
// straight into fragments, two lines at a time.  KS = 1: a wave has 32 rows to itself, which halves what it reads of F.  KS = 4, for few
// rows: four waves split the lines of 16 rows, their sums meet in LDS.  g.turns workgroups share a tile's models in turn (one model's product is
// a chain of loads of some microseconds); the first of them clears what no model owns.
// In a pass, with the layout that rides along: 65,536 rows of 1,024 bf16 of 16 models 43 us (35 the fastest, 134 MB: 3.8 TB/s), 2,048 rows fp32
// 10 us (8.7), 61 rows of 512 fp32 6.6 us.
template <int RT, int KS> constexpr int kShrinkLds = KS > 1 ? KS * RT * 4 * 64 : 1;  // floats
template <typename T, int RT, int KS>
__device__ void shrink_body(const ShrinkArgs& g, unsigned block, int j0, const T* __restrict__ x, const T* __restrict__ F, Low<T>* __restrict__ u, Low<T>* __restrict__ uT, float* lds) {
    constexpr int V = mtk_piece<T>::n, KB = kLine<T>, RR = KS > 1 ? 1 : 2;
    float (*part)[KS > 1 ? RT * 4 : 1][64] = reinterpret_cast<float (*)[KS > 1 ? RT * 4 : 1][64]>(lds);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, q = lane >> 4;
    const int my_turn = block / (unsigned)g.tiles;  // neighbours go to different XCDs, so the turns must not alternate
    const int64_t m0 = ((int64_t)(block % (unsigned)g.tiles) * (4 / KS) + (KS > 1 ? 0 : wave)) * 16 * RR;
    if (m0 >= g.M) return;
    const int64_t end = m0 + 16 * RR < g.M ? m0 + 16 * RR : g.M;
    const T* xr[RR];
#pragma unroll
    for (int p = 0; p < RR; ++p) xr[p] = x + (m0 + p * 16 + li < g.M ? m0 + p * 16 + li : g.M - 1) * g.x_ld + q * V;
    f32x4 keep[RR][RT] = {};
    bool mine[RR] = {}, any[RR] = {};  // this lane's rows: computed here / owned by any model
    int who[RR];
#pragma unroll
    for (int p = 0; p < RR; ++p) who[p] = -1;
    Owners own(g.offsets, g.E, m0, end);
    int e, turn = 0;
    int64_t a, b;
    while (own.next(e, a, b)) {
        bool in[RR];
#pragma unroll
        for (int p = 0; p < RR; ++p) {
            in[p] = m0 + p * 16 + li >= a && m0 + p * 16 + li < b;
            any[p] |= in[p];
            who[p] = in[p] ? e : who[p];
        }
        if (turn++ % g.turns != my_turn) continue;
#pragma unroll
        for (int p = 0; p < RR; ++p) mine[p] |= in[p];
        const T* fr[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int j = j0 + t * 16 + li;
            fr[t] = F + ((int64_t)e * g.r + (j < g.r ? j : g.r - 1)) * g.K + q * V;
        }
        f32x4 acc[RR][RT] = {};
        const int step = KS > 1 ? KS * KB : KB;
        int k0 = KS > 1 ? wave * KB : 0;
        auto lines = [&](auto count) {
            constexpr int L = decltype(count)::value;
            mtk_vec<T> xv[L][RR][2], fv[L][RT][2];
#pragma unroll
            for (int l = 0; l < L; ++l) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int p = 0; p < RR; ++p) xv[l][p][h] = mtk_ld(xr[p] + k0 + l * step + h * 4 * V);
#pragma unroll
                    for (int t = 0; t < RT; ++t) fv[l][t][h] = mtk_ld(fr[t] + k0 + l * step + h * 4 * V);
                }
            }
#pragma unroll
            for (int l = 0; l < L; ++l)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int p = 0; p < RR; ++p)
#pragma unroll
                        for (int t = 0; t < RT; ++t) acc[p][t] = mma16(fv[l][t][h], xv[l][p][h], acc[p][t]);
            k0 += L * step;
        };
        constexpr int U = RT == 4 ? 2 : (KS > 1 && RT == 1 ? 8 : 4);
        while (k0 + (U - 1) * step + KB <= g.K) lines(std::integral_constant<int, U>());
        while (k0 + KB <= g.K) lines(std::integral_constant<int, 1>());
        if (k0 < g.K) {  // the last, partial line
            const int left = g.K - k0 - q * V;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    const mtk_vec<T> f = mtk_ld_n(fr[t] + k0 + h * 4 * V, left - h * 4 * V);
#pragma unroll
                    for (int p = 0; p < RR; ++p) acc[p][t] = mma16(f, mtk_ld_n(xr[p] + k0 + h * 4 * V, left - h * 4 * V), acc[p][t]);
                }
        }
        if (KS > 1) {
            __syncthreads();
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) part[wave][t * 4 + i][lane] = acc[0][t][i];
            __syncthreads();
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v = 0.f;
#pragma unroll
                    for (int w = 0; w < KS; ++w) v += part[w][t * 4 + i][lane];
                    acc[0][t][i] = v;
                }
        }
        const float s = g.scales ? g.scales[e] : g.scale;
#pragma unroll
        for (int p = 0; p < RR; ++p)
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) keep[p][t][i] = in[p] ? s * acc[p][t][i] : keep[p][t][i];
    }
    if (KS > 1 && wave > 0) return;
    TileModels tm = {};
    const int tile = g.BM > 0 ? (int)(m0 / g.BM) : 0;  // 64 rows or more: all of this wave's are in it
    if (g.BM > 0) tm = TileModels::of_tile(own, (int64_t)tile * g.BM, g.BM, g.M, g.E);
#pragma unroll
    for (int p = 0; p < RR; ++p) {
        if (!(mine[p] || (my_turn == 0 && !any[p]))) continue;  // a row without a model: zeros
        const int64_t at = m0 + p * 16 + li;  // D[j][record]: lane & 15 -> record, j = 4 (lane >> 4) + register
        typedef Low<T> L;
        constexpr int P = kParts<T>, S = kSections<T>;
        struct __attribute__((aligned(4 * sizeof(L)), may_alias)) Quad { L v[4]; };
        const int sec = section<T>(g.r);
        const int64_t plane = mtk_up(g.r, 64) * g.Mp;  // of u^T: a number each
        L* ur = u + at * g.rp;
        auto put = [&](L* row, const Quad (&o)[P], bool its) {
#pragma unroll
            for (int c = 0; c < S; ++c) *reinterpret_cast<Quad*>(row + c * sec) = its ? o[section_part(c)] : Quad{};
        };
        auto pair_row = [&](int i) { return (L*)g.pairs + ((int64_t)(tile + tm.e + i) * g.BM + (at - (int64_t)tile * g.BM)) * g.rp; };
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            Quad o[P];
            const int j = j0 + t * 16 + q * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                L n[P];
                parts_of(j + i < g.r ? keep[p][t][i] : 0.f, n);
#pragma unroll
                for (int c = 0; c < P; ++c) o[c].v[i] = n[c];
            }
            if (at < g.M && j < sec) {
                put(ur + j, o, true);
                if (tm.ranged)
                    for (int i = 0; i < tm.count; ++i) put(pair_row(i) + j, o, tm.e + i == who[p]);
            }
            if (uT && at < g.Mp)  // mtk_up(r, 64) rows of Mp
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int c = 0; c < P; ++c) uT[c * plane + (int64_t)(j + i) * g.Mp + at] = o[c].v[i];
        }
        if (j0 + RT * 16 >= g.r && at < g.M) {  // zeros up to the end of the sections, and of the row
            const Quad zero[P] = {};
            for (int j = j0 + RT * 16 + q * 4; j < sec; j += 16) {
                put(ur + j, zero, true);
                if (tm.ranged)
                    for (int i = 0; i < tm.count; ++i) put(pair_row(i) + j, zero, true);
            }
            if constexpr (kF16<T>)
                for (int j = S * sec + q * 4; j < g.rp; j += 16) {
                    *reinterpret_cast<Quad*>(ur + j) = Quad{};
                    if (tm.ranged)
                        for (int i = 0; i < tm.count; ++i) *reinterpret_cast<Quad*>(pair_row(i) + j) = Quad{};
                }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------ linear
// y = act(x W^T + b + u B_e^T).  Weights are the MFMA's A operand: a lane then holds consecutive features of one record.
//
// k_linear, for more than a few rows: persistent workgroups walk tiles of BM rows x BN features; the k-blocks of ALL their tiles form one
// stream of LDS-DMA (DX buffers for rows, DW for weights), so a tile's epilogue runs with the next tile's first blocks in flight.
// The low-rank product is the last k-blocks of a tile: rows of u against rows of B_e (both zero behind the rank), the same
// instructions through the same buffers.  A tile that several models share, or some rows of which have none, takes these blocks once
// per model e from the tile's pair (t, e) of rows, in which the other models' are zero.  Walking the tiles, each step to the next pair raises t, e or
// both, so t + e numbers the pairs.  Zero times B_e is zero while B_e is finite; a shared tile with one that is not is made once more, without
// the stream.  There, in tiles of more than kTileModels models, and (nkx = 0) with far fewer rows a model than a tile has, the
// low-rank products are made in the epilogue, per model, and selected by row.
// 65,536 x 1,024 x 1,024 in bf16, in a pass, 161 us (146 the fastest), 17 lines of k for the 16 of the shared product alone, which the library's plain
// product does in 133; 2,048 rows in fp32 51 us (48.5; 33 lines for 32; 35): there the matrix pipes are busy 69 % of the kernel's cycles, the
// rest is start, end and a barrier a line.
// RAW, fp16 without such blocks: B_e as it lies, split into its two numbers where it is read (a kernel of its own: with the lines' loop beside
// it the accumulators spill; lines for all would be laid out at length: 2,048 rows of 128 models 58 us for 20).
// The stream wants whole, 16-byte aligned lines: k_prep pads what is not, and lays out B, the bias in fp32, the tiles' models and which B_e
// hold infinities or NaN.
struct LinearArgs {
    int64_t M, MT;        // rows, row tiles
    int N, nb_n;          // features, feature tiles
    int nkb, nkx;         // k-blocks of the shared and of the low-rank product
    int64_t x_ld, w_ld;   // row strides, in bytes
    const void *X, *W, *U, *Bp;  // U [M][nkx lines], Bp [E][N][nkx lines]
    const void* pairs;    // [MT + E][BM][nkx lines]
    void* Y;
    const float* bias;    // [nb_n * BN]
    const int32_t* owner; // [MT] TileModels
    const int32_t* odd;   // [E] not 0: B_e holds infinities or NaN
    const int32_t* offsets;
    int E, relu;
    const void* low;      // [E][N][low_ld] B_e for the epilogue, in whole pieces, zeros behind the rank
    int low_ld, rp, r;    // rp: elements of a row of U
};

// WR x WC waves, each MW x NT tiles of 32 x 32; DX buffers of rows and DW of weights
template <int WR, int WC_, int MW, int NT, int DX_, int DW_> struct Geo {
    static constexpr int WC = WC_, NW = WR * WC, WN = NT * 32, BM = WR * MW * 32, BN = WC * WN;
    static constexpr int kTileX = BM * 128, kTileW = BN * 128;       // bytes of a k-block
    static constexpr int XPW = BM / 8 / NW, WPW = BN / 8 / NW;       // 8-row, 1 KiB pieces per wave
    static constexpr int DX = DX_, DW = DW_, kLds = DX * kTileX + DW * kTileW;
    static constexpr int kRoom = 163840 / kLds, kWaves = kRoom * NW / 4;  // workgroups of a CU, waves of a SIMD: a register too many halves them
    static constexpr int kYounger = XPW + (DW - 2) * (XPW + WPW);    // pieces a wave requests after its last of the next block
};

extern __shared__ __attribute__((aligned(16))) unsigned char ad_smem[];

// The arguments, read anew where they are used: the work between two tiles needs them all, and kept in scalar registers over the k-blocks (or
// spilled to lanes of vector registers) they would be paid for in every one.
typedef const __attribute__((address_space(4))) LinearArgs KernelArgs;
__device__ __forceinline__ KernelArgs& linear_args() {
    auto p = __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(KernelArgs*)p;
}

// a uniform value through the scalar cache: a vector load would wait for all the DMA requested before it
__device__ __forceinline__ int scalar_load(const int32_t* p) {
    int v;
    asm volatile("s_load_dword %0, %1, 0x0\n\ts_waitcnt lgkmcnt(0)" : "=&s"(v) : "s"(p) : "memory");
    return v;
}

template <typename T, int WR, int WC, int MW, int NT, int DX, int DW, bool RAW>
__global__ __launch_bounds__(64 * WR * WC, (Geo<WR, WC, MW, NT, DX, DW>::kWaves)) void k_linear(LinearArgs) {  // (linear_args)
    typedef Geo<WR, WC, MW, NT, DX, DW> G;
    constexpr int V = mtk_piece<T>::n, kWBase = DX * G::kTileX;
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const int wv = __builtin_amdgcn_readfirstlane(wid);
    const int wr = wv / WC, wc = wv % WC, li = lane & 31, hh = lane >> 5;
    // workgroups go round-robin over the 8 XCDs: each XCD takes a contiguous eighth of the tiles (features fastest), so a row tile's
    // feature tiles run side by side on one XCD's L2 and every XCD has work
    const int xcd = blockIdx.x & 7, wq = blockIdx.x >> 3, wstride = gridDim.x >> 3;
    KernelArgs& first_args = linear_args();
    const int nb_n = first_args.nb_n, tiles = (int)first_args.MT * nb_n, per = (tiles + 7) / 8, first = xcd * per;
    const int slots = tiles - first < per ? tiles - first : per;
    if (wq >= slots) return;
    // DMA of one 8-row piece (64 lanes x 16 bytes): lane -> row lane >> 3, piece slot lane & 7.  The LDS image is linear in the lane, so the
    // bank swizzle (slot s of row r holds piece s ^ ((r >> 1) & 7)) is applied to the global address.  Rows behind the last are
    // clamped: they are read again, never stored.  M0 (the LDS address) is written with every piece; the compiler puts nothing there.
    // A cursor keeps what its next block needs: a scalar base that moves on by a line a block, and the wave's piece offsets, worked out
    // anew when the source changes (a tile's operand, then its low-rank lines).
    const int lr = lane >> 3, lc0 = ((lane & 7) ^ (lr >> 1)) * 16, lc1 = ((lane & 7) ^ ((lr >> 1) | 4)) * 16;
    auto offsets = [&](unsigned* voff, int n, int chunk0, int rows, unsigned ld) {
#pragma unroll
        for (int j = 0; j < n; ++j) {
            const int rr = (chunk0 + j) * 8 + lr, rc = rr < rows ? rr : rows - 1;
            voff[j] = (unsigned)rc * ld + (unsigned)((chunk0 + j) & 1 ? lc1 : lc0);
        }
    };
    auto dma = [&](const unsigned char* gp, unsigned voff, unsigned dst) {
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(voff), "s"(gp), "s"(dst) : "memory");
    };
    // The common step of a cursor is an addition, a wrap and a countdown: with one or two waves on a SIMD, scalar work between two
    // barriers is time.
    const unsigned x_dst0 = (unsigned)(wv * G::XPW * 1024), w_dst0 = (unsigned)(kWBase + wv * G::WPW * 1024);
    unsigned x_dst = x_dst0, w_dst = w_dst0;
    int cx_slot = wq, cw_slot = wq, x_left = 0, w_left = 0;  // blocks left at the source
    int x_low = 1, w_low = 1;  // 1: the source is the low-rank lines (an int: a bool that loops is kept as a lane mask, and its selects in vector registers)
    const unsigned char *xb = nullptr, *wb = nullptr;
    unsigned xoff[G::XPW], woff[G::WPW];
    int x_more = 0, w_more = 0;  // models of the tile still to come
    auto x_source = [&]() {  // the next source of the row cursor; none: never counts down again
        KernelArgs& g = linear_args();
        const unsigned lo_ld = (unsigned)g.nkx * 128;
        if (x_more > 0) {  // from behind this pair's lines to the next pair's
            --x_more;
            x_left = g.nkx;
            xb += (int64_t)(G::BM - 1) * lo_ld;
            return;
        }
        TileModels m = {0, 0, 0, 0};
        if (x_low == 0 && g.nkx > 0) m = TileModels::of(scalar_load(g.owner + (first + cx_slot) / nb_n));
        x_low = m.count > 0 ? 1 : 0;
        if (x_low == 0) {
            if (x_left < 0) cx_slot += wstride;
            if (cx_slot >= slots) {
                x_left = 0x7fffffff;
                return;
            }
        }
        const int mt = (first + cx_slot) / nb_n;
        const int64_t m0 = (int64_t)mt * G::BM;
        const int rows = g.M - m0 < G::BM ? (int)(g.M - m0) : G::BM;
        unsigned ld;
        if (x_low) {
            x_left = g.nkx;
            x_more = m.count - 1;
            xb = m.ranged ? (const unsigned char*)g.pairs + (int64_t)(mt + m.e) * G::BM * lo_ld : (const unsigned char*)g.U + m0 * lo_ld;
            ld = lo_ld;
        } else {
            x_left = g.nkb;
            xb = (const unsigned char*)g.X + m0 * g.x_ld;
            ld = (unsigned)g.x_ld;
        }
        offsets(xoff, G::XPW, wv * G::XPW, rows, ld);
    };
    auto w_source = [&]() {
        KernelArgs& g = linear_args();
        const unsigned lo_ld = (unsigned)g.nkx * 128;
        if (w_more > 0) {  // from behind this model's lines to the next model's
            --w_more;
            w_left = g.nkx;
            wb += (int64_t)(g.N - 1) * lo_ld;
            return;
        }
        TileModels m = {0, 0, 0, 0};
        if (w_low == 0 && g.nkx > 0) m = TileModels::of(scalar_load(g.owner + (first + cw_slot) / nb_n));
        w_low = m.count > 0 ? 1 : 0;
        if (w_low == 0) {
            if (w_left < 0) cw_slot += wstride;
            if (cw_slot >= slots) {
                w_left = 0x7fffffff;
                return;
            }
        }
        const int id = first + cw_slot, mt = id / nb_n, n0 = (id - mt * nb_n) * G::BN;
        const int rows = g.N - n0 < G::BN ? g.N - n0 : G::BN;
        unsigned ld;
        if (w_low) {
            w_left = g.nkx;
            w_more = m.count - 1;
            wb = (const unsigned char*)g.Bp + ((int64_t)m.e * g.N + n0) * lo_ld;
            ld = lo_ld;
        } else {
            w_left = g.nkb;
            wb = (const unsigned char*)g.W + (int64_t)n0 * g.w_ld;
            ld = (unsigned)g.w_ld;
        }
        offsets(woff, G::WPW, wv * G::WPW, rows, ld);
    };
    auto x_op = [&](int j) {
        if (cx_slot < slots) dma(xb, xoff[j], x_dst + j * 1024);
    };
    auto w_op = [&](int j) {
        if (cw_slot < slots) dma(wb, woff[j], w_dst + j * 1024);
    };
    auto x_advance = [&]() {
        xb += 128;
        x_dst = x_dst == x_dst0 + (DX - 1) * G::kTileX ? x_dst0 : x_dst + G::kTileX;
        if (--x_left == 0) {
            x_left = -1;
            x_source();
        }
    };
    auto w_advance = [&]() {
        wb += 128;
        w_dst = w_dst == w_dst0 + (DW - 1) * G::kTileW ? w_dst0 : w_dst + G::kTileW;
        if (--w_left == 0) {
            w_left = -1;
            w_source();
        }
    };
    const unsigned char* lds = ad_smem;
    struct Frags { mtk_vec<T> x[MW], w[NT]; };
    auto read_frags = [&](Frags& f, int xi, int wi, int ks) {
#pragma unroll
        for (int q = 0; q < MW; ++q) {
            const int ra = (wr * MW + q) * 32 + li, kp = ks * 2 + hh;
            f.x[q] = __builtin_bit_cast(mtk_vec<T>, *reinterpret_cast<const uint4*>(lds + xi * G::kTileX + ra * 128 + ((kp ^ ((ra >> 1) & 7)) * 16)));
        }
#pragma unroll
        for (int q = 0; q < NT; ++q) {
            const int rb = wc * G::WN + q * 32 + li, kp = ks * 2 + hh;
            f.w[q] = __builtin_bit_cast(mtk_vec<T>, *reinterpret_cast<const uint4*>(lds + kWBase + wi * G::kTileW + rb * 128 + ((kp ^ ((rb >> 1) & 7)) * 16)));
        }
    };
    f32x16 acc[MW][NT];
    auto mma_row = [&](auto type, const Frags& f, int mt) {  // type: of the numbers in the fragments
        typedef mtk_vec<decltype(type)> F;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = mma32(__builtin_bit_cast(F, f.w[nt]), __builtin_bit_cast(F, f.x[mt]), acc[mt][nt]);
    };
    auto mma_all = [&](auto type, const Frags& f) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int mt = 0; mt < MW; ++mt) mma_row(type, f, mt);
        __builtin_amdgcn_sched_barrier(0);
    };

    // One k-block: four steps of two pieces, fragments read one step ahead.  The barrier sits before the last step's MFMAs; the fragment reads
    // and the DMA requests behind it ride under them.  After the barrier of block c a wave requests its pieces of weight block c + DW,
    // THEN of row block c + DX (DX >= DW).  Loads return in order, so at the end of block c all but the kYounger pieces requested after
    // weight block c + 1 (row block c + 1 is older still) done means that block c + 1 has landed.
    // the accumulators start from the bias, through the SCALAR cache: vector loads here would queue behind the DMA in flight
    auto start = [&](int n0) {
        const float* bp = linear_args().bias + n0 + wc * G::WN;
#pragma unroll
        for (int h = 0; h < 2 * NT; ++h) {  // 16 features at a time: more would spill scalar registers
            f32x8 b0, b1;
            asm volatile("s_load_dwordx8 %0, %2, 0x0\n\ts_load_dwordx8 %1, %2, 0x20\n\ts_waitcnt lgkmcnt(0)" : "=&s"(b0), "=&s"(b1) : "s"(bp + h * 16) : "memory");
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float v0 = hh ? b0[4 + j] : b0[j], v1 = hh ? b1[4 + j] : b1[j];
#pragma unroll
                for (int a = 0; a < MW; ++a) {
                    acc[a][h >> 1][8 * (h & 1) + j] = v0;
                    acc[a][h >> 1][8 * (h & 1) + 4 + j] = v1;
                }
            }
        }
    };

    Frags F0, F1;
    x_source();
    w_source();
    for (int b = 0; b < DX; ++b) {
#pragma unroll
        for (int j = 0; j < G::XPW; ++j) x_op(j);
        x_advance();
        if (b < DW) {
#pragma unroll
            for (int j = 0; j < G::WPW; ++j) w_op(j);
            w_advance();
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int xi = 0, wi = 0;   // buffers of the block being consumed
    bool x_tail = false;  // the previous block's tail requested row pieces after its weight pieces
    for (int slot = wq; slot < slots; slot += wstride) {
        const int id = first + slot, mtile = id / nb_n, n0 = (id - mtile * nb_n) * G::BN;
        const int64_t m0 = (int64_t)mtile * G::BM;
        KernelArgs& ga = linear_args();
        const int tm = ga.nkx ? scalar_load(ga.owner + mtile) : 0;
        const int nk = ga.nkb + ga.nkx * TileModels::of(tm).count;
        start(n0);
        read_frags(F0, xi, wi, 0);
        // Stores of the previous tile may be outstanding too and do not return in order with the loads, but the count still holds: with S stores,
        // N needed and kYounger younger pieces in flight, "at most kYounger outstanding" needs S + N completions, and fewer than
        // N loads done (the needed ones come first) would leave at most S + N - 1.
        // (The barrier: everyone's share has landed, and this block's buffers have no readers left.)  A macro: as a lambda, whose captures are kept
        // differently, the same lines cost fp32 3 % (2,048 rows 52.1 -> 54.3 us).
#define MTK_BLOCKS(TYPE, FROM, TO) \
        for (int kb = FROM; kb < TO; ++kb) { \
            read_frags(F1, xi, wi, 1); \
            mma_all(TYPE, F0); \
            read_frags(F0, xi, wi, 2); \
            mma_all(TYPE, F1); \
            read_frags(F1, xi, wi, 3); \
            mma_all(TYPE, F0); \
            if (x_tail) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(G::kYounger) : "memory"); \
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); \
            __syncthreads(); \
            __builtin_amdgcn_sched_barrier(0); \
            const int xn = xi == DX - 1 ? 0 : xi + 1, wn = wi == DW - 1 ? 0 : wi + 1; \
            if (kb + 1 < nk) read_frags(F0, xn, wn, 0); \
            constexpr int OPW = G::XPW + G::WPW; \
_Pragma("unroll") \
            for (int mt = 0; mt < MW; ++mt) { \
                __builtin_amdgcn_sched_barrier(0); \
                mma_row(TYPE, F1, mt); \
                __builtin_amdgcn_sched_barrier(0); \
_Pragma("unroll") \
                for (int j = mt * OPW / MW; j < (mt + 1) * OPW / MW; ++j) { \
                    if (j < G::WPW) w_op(j); \
                    else x_op(j - G::WPW); \
                } \
            } \
            w_advance(); \
            x_tail = cx_slot < slots; \
            x_advance(); \
            xi = xn; \
            wi = wn; \
            __builtin_amdgcn_sched_barrier(0); \
        }
        if constexpr (kF16<T> && !RAW) {  // the low-rank blocks hold other numbers
            MTK_BLOCKS(T(0), 0, ga.nkb)
            MTK_BLOCKS(Low<T>(0), ga.nkb, nk)
        } else {
            MTK_BLOCKS(T(0), 0, nk)
        }
#undef MTK_BLOCKS

        // opaque copy of the lane id: what the epilogue derives from it is recomputed per tile instead of being kept alive across the k-loop
        int lane_e = lane;
        asm volatile("" : "+v"(lane_e));
        const int li_e = lane_e & 31, hh_e = lane_e >> 5;
        KernelArgs& g = linear_args();
        T* const __restrict__ y = (T*)g.Y;
        int apart = !g.nkx || TileModels::of(tm).many;  // the low-rank products are still to come
        if (TileModels::of(tm).ranged) {
            int odd = 0;
            for (int i = 0; i < TileModels::of(tm).count; ++i) odd |= scalar_load(g.odd + TileModels::of(tm).e + i);
            if (odd) {  // 0 x inf has been in it: once more, straight from memory, the same products in the same order
                apart = 1;
                start(n0);
#pragma unroll 1
                for (int kp = hh_e * 16; kp < g.nkb * 128; kp += 32) {
                    Frags f;
#pragma unroll
                    for (int q = 0; q < MW; ++q) {
                        const int64_t row = m0 + (wr * MW + q) * 32 + li_e;
                        f.x[q] = mtk_ld((const T*)((const char*)g.X + (row < g.M ? row : g.M - 1) * g.x_ld + kp));
                    }
#pragma unroll
                    for (int q = 0; q < NT; ++q) {
                        const int n = n0 + wc * G::WN + q * 32 + li_e;
                        f.w[q] = mtk_ld((const T*)((const char*)g.W + (int64_t)(n < g.N ? n : g.N - 1) * g.w_ld + kp));
                    }
                    mma_all(T(0), f);
                }
            }
        }
        if (g.low && apart) {
            const int64_t w0 = m0 + wr * MW * 32, w1 = w0 + MW * 32;
            Owners own(g.offsets, g.E, w0, w1 < g.M ? w1 : g.M);
            int e;
            int64_t a, b;
            typedef Low<T> L;
            const L* u = (const L*)g.U;
            constexpr int S = 32 / (2 * V);  // steps of 32 values of the rank
            const int sec = section<T>(g.r), low_n = kF16<T> || g.low_ld < sec ? g.low_ld : sec;  // B_e's values, once
            while (own.next(e, a, b)) {
                const T* be = (const T*)g.low + (int64_t)e * g.N * g.low_ld;
#pragma unroll
                for (int mt = 0; mt < MW; ++mt) {
                    const int64_t row = w0 + mt * 32 + li_e, rc = row < g.M ? row : g.M - 1;
                    const bool mine = row >= a && row < b;
                    if (a >= w0 + mt * 32 + 32 || b <= w0 + mt * 32) continue;
                    const L* ur = u + rc * g.rp;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const int n = n0 + wc * G::WN + nt * 32 + li_e;
                        f32x16 low = acc[mt][nt];
                        if constexpr (kF16<T> && !RAW) {  // whole lines against whole lines, in the stream's order: a row that is made once more keeps its bits
                            const L* bn = (const L*)be + (int64_t)(n < g.N ? n : g.N - 1) * g.low_ld;
#pragma unroll 1
                            for (int k = hh_e * V; k < g.rp; k += 2 * V * S) {
                                mtk_vec<L> uv[S], bv[S];  // requested together: one round trip
#pragma unroll
                                for (int s = 0; s < S; ++s) {
                                    uv[s] = mtk_ld(ur + k + s * 2 * V);
                                    bv[s] = mtk_ld(bn + k + s * 2 * V);
                                }
#pragma unroll
                                for (int s = 0; s < S; ++s) low = mma32(bv[s], uv[s], low);
                            }
                        } else {
                            auto piece = [&](int j) {  // of B_e, zeros behind the rank
                                const bool in = j < low_n;
                                const uint4 w = __builtin_bit_cast(uint4, mtk_ld(be + mtk_low_piece(n, g.N, g.low_ld, low_n, j)));
                                return __builtin_bit_cast(mtk_vec<T>, make_uint4(in ? w.x : 0u, in ? w.y : 0u, in ? w.z : 0u, in ? w.w : 0u));
                            };
                            if constexpr (kF16<T>) {
#pragma unroll 1
                                for (int j = hh_e * V; j < g.r + hh_e * V; j += 2 * V) {  // (what is behind a section of u meets zeros)
                                    const mtk_vec<T> bt = piece(j);
                                    const mtk_vec<L> u0 = mtk_ld(ur + j), u1 = mtk_ld(ur + sec + j), u2 = mtk_ld(ur + 2 * sec + j);
                                    mtk_vec<L> bv = number_of(bt, false);
                                    low = mma32(bv, u2, low);
                                    low = mma32(bv, u1, low);
                                    low = mma32(bv, u0, low);
                                    bv = number_of(bt, true);
                                    low = mma32(bv, u1, low);
                                    low = mma32(bv, u0, low);
                                }
                            } else {
                                auto steps = [&](int j0, int h, auto count) {  // requested together: one round trip
                                    constexpr int C = decltype(count)::value;
                                    mtk_vec<T> uv[C], bv[C];
#pragma unroll
                                    for (int s = 0; s < C; ++s) {
                                        const int j = j0 + s * 2 * V;
                                        bv[s] = piece(j + hh_e * V);
                                        uv[s] = mtk_ld(ur + h + j + hh_e * V);
                                    }
#pragma unroll
                                    for (int s = 0; s < C; ++s) low = mma32(bv[s], uv[s], low);
                                };
#pragma unroll 1
                                for (int h = 0; h < g.rp; h += sec)
#pragma unroll 1
                                    for (int j0 = 0; j0 < g.r; j0 += 32) steps(j0, h, std::integral_constant<int, S>());
                            }
                        }
#pragma unroll
                        for (int q = 0; q < 16; ++q) acc[mt][nt][q] = mine ? low[q] : acc[mt][nt][q];
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
#pragma unroll
        for (int mt = 0; mt < MW; ++mt) {
            const int64_t row = m0 + (wr * MW + mt) * 32 + li_e;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if (g.relu) {
#pragma unroll
                    for (int q = 0; q < 16; ++q) acc[mt][nt][q] = acc[mt][nt][q] < 0.f ? 0.f : acc[mt][nt][q];  // NaN stays
                }
                const int nb = n0 + wc * G::WN + nt * 32;
                if constexpr (sizeof(T) == 4) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int n = nb + 8 * q + 4 * hh_e;
                        mtk_vec<T> o;
#pragma unroll
                        for (int j = 0; j < 4; ++j) o.v[j] = acc[mt][nt][4 * q + j];
                        if (row < g.M) {
                            if (n + 4 <= g.N) mtk_st(y + row * g.N + n, o);
                            else mtk_st_n(y + row * g.N + n, o, g.N - n);
                        }
                    }
                } else {
                    // lanes l and l + 32 hold the two halves of every 8-feature piece: v_permlane32_swap gives each a whole 16-byte piece
#pragma unroll
                    for (int p2 = 0; p2 < 2; ++p2) {
                        unsigned pk[2][2];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            T h[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) h[j] = (T)acc[mt][nt][4 * (2 * p2 + i) + j];
                            pk[i][0] = reinterpret_cast<const unsigned*>(h)[0];
                            pk[i][1] = reinterpret_cast<const unsigned*>(h)[1];
                        }
                        const auto r0 = __builtin_amdgcn_permlane32_swap(pk[1][0], pk[0][0], false, false);
                        const auto r1 = __builtin_amdgcn_permlane32_swap(pk[1][1], pk[0][1], false, false);
                        const int n = nb + 8 * (2 * p2 + (hh_e ? 0 : 1));
                        const mtk_vec<T> o = __builtin_bit_cast(mtk_vec<T>, make_uint4(r0[0], r1[0], r0[1], r1[1]));
                        if (row < g.M) {
                            if (n + 8 <= g.N) mtk_st(y + row * g.N + n, o);
                            else mtk_st_n(y + row * g.N + n, o, g.N - n);
                        }
                    }
                }
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// k_linear_few, for few rows: bound by the latency of streaming W once.  TS rows x TS features a workgroup (16 up to 64 rows, else 32), its eight
// waves split k and take their fragments straight from memory; partial sums meet in LDS.  The low-rank product is plain FMAs there, each row
// with its own model.  61 rows of 512 to 1,024 features fp32 5.5 us.
// What the end needs (offsets, bias, the low-rank operands) is requested between the first lines' loads and their
// products: each would be a round trip of its own otherwise.
// FUSED, for a row or some (M r <= kFusedPairs): every workgroup computes u itself, a wave a value at a time, under W's loads; the first writes it
// for the backward.  One launch for two, whose own time is, fused / apart, in us: one row of 1,024 at rank 8 in bf16 7.3 / 6.2 + 3.8, at rank
// 32 10.8 / 6.8 + 5.1, sixteen of 512 at rank 2 in fp32 9.5 / 6.0 + 4.8; four values at a time 15 for the first.
constexpr int kFusedPairs = 32;
struct FewArgs {
    int64_t M, x_ld;
    int N, K, r, rp, E, relu;
    const int32_t* offsets;
    const float* scales;  // FUSED from here on
    float scale;
    int64_t Mp;
};

template <typename T, int TS, bool FUSED>
__global__ __launch_bounds__(512) void k_linear_few(FewArgs g, const T* __restrict__ x, const T* __restrict__ W, const T* __restrict__ bias, const Low<T>* __restrict__ u,
                                                    const T* __restrict__ up, T* __restrict__ y, const T* __restrict__ down, Low<T>* __restrict__ u_out, Low<T>* __restrict__ uT) {
    typedef Low<T> L;
    constexpr int V = mtk_piece<T>::n, KB = kLine<T>, NW = 8;
    constexpr int LANES = 64 / TS, S = 8 / LANES;  // lanes that share a row, steps of a line
    constexpr int OUT = TS * TS > 512 ? 2 : 1;     // outputs of a thread
    typedef typename std::conditional<TS == 32, f32x16, f32x4>::type Acc;
    __shared__ float part[NW][TS][TS + 1];
    __shared__ float us[FUSED ? kFusedPairs : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & (TS - 1), hh = lane / TS;
    const int nb = (g.N + TS - 1) / TS;
    const int64_t m0 = (int64_t)(blockIdx.x / nb) * TS;
    const int n0 = (int)(blockIdx.x % nb) * TS;
    const T* xr = x + (m0 + li < g.M ? m0 + li : g.M - 1) * g.x_ld + hh * V;
    const T* wr = W + (int64_t)(n0 + li < g.N ? n0 + li : g.N - 1) * g.K + hh * V;
    auto mma = [](const mtk_vec<T>& a, const mtk_vec<T>& b, Acc c) {
        if constexpr (TS == 32) return mma32(a, b, c);
        else return mma16(a, b, c);
    };
    const int held = lane <= g.E ? g.offsets[lane] : 0x7fffffff;
    // the wave's first two lines, zeros where there are none
    mtk_vec<T> xa[2][S], wa[2][S];
#pragma unroll
    for (int l = 0; l < 2; ++l) {
        const int k0 = (wave + l * NW) * KB;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int k = k0 + s * LANES * V, left = g.K - k - hh * V;
            if (k0 + KB <= g.K) {
                xa[l][s] = mtk_ld(xr + k);
                wa[l][s] = mtk_ld(wr + k);
            } else {
                xa[l][s] = mtk_ld_n(xr + k, left);
                wa[l][s] = mtk_ld_n(wr + k, left);
            }
        }
    }
    // this thread's outputs: row rr + 16 i, feature n; models by ballots over the offsets
    const int rr = tid / TS, n = n0 + (tid & (TS - 1)), nc = n < g.N ? n : g.N - 1;
    constexpr int LP = 16 / V;  // pieces of the rank requested ahead: 16 values
    constexpr int H = kParts<T>;  // numbers of a value of u, in the first sections
    const int sec = section<T>(g.r);
    auto value = [](const mtk_vec<L> (&v)[H], int c) {
        float f = (float)v[0].v[c];
#pragma unroll
        for (int h = 1; h < H; ++h) f += (float)v[h].v[c];
        return f;
    };
    const float bv = bias ? (float)bias[nc] : 0.f;
    int who[OUT];
    mtk_vec<L> ua[OUT][LP][H];
    mtk_vec<T> ba[OUT][LP];
#pragma unroll
    for (int i = 0; i < OUT; ++i) {
        const int64_t row = m0 + rr + 16 * i, rc = row < g.M ? row : g.M - 1;
        int c = 0;
#pragma unroll
        for (int q = 0; q < LANES; ++q) {  // the wave's rows
            const int64_t at = m0 + wave * LANES + q + 16 * i;
            int cq = __popcll(__ballot(held <= at));
            for (int e0 = 64; e0 <= g.E; e0 += 64) cq += __popcll(__ballot((e0 + lane <= g.E ? g.offsets[e0 + lane] : 0x7fffffff) <= at));
            c = hh == q ? cq : c;
        }
        who[i] = c - 1;
        if (who[i] < 0 || who[i] >= g.E || row >= g.M || rr + 16 * i >= TS) who[i] = -1;
        const L* ur = u + rc * g.rp;
        const T* br = up + ((int64_t)(who[i] < 0 ? 0 : who[i]) * g.N + nc) * g.r;
#pragma unroll
        for (int p = 0; p < LP; ++p) {
#pragma unroll
            for (int h = 0; h < H; ++h)
                if (!FUSED) ua[i][p][h] = mtk_ld(ur + h * sec + p * V);  // inside the row, which is whole lines; up's zeros behind the rank
            ba[i][p] = p * V + V <= g.r ? mtk_ld(br + p * V) : mtk_ld_n(br + p * V, g.r - p * V);
        }
    }
    if constexpr (FUSED) {
        for (int q = wave; q < (int)g.M * g.r; q += NW) {
            const int row = q / g.r, j = q - row * g.r;
            int c = __popcll(__ballot(held <= row));
            for (int e0 = 64; e0 <= g.E; e0 += 64) c += __popcll(__ballot((e0 + lane <= g.E ? g.offsets[e0 + lane] : 0x7fffffff) <= row));
            const int e = c - 1;
            float v = 0.f;
            if (e >= 0 && e < g.E) {
                const T *xp = x + row * g.x_ld, *ap = down + ((int64_t)e * g.r + j) * g.K;
                for (int k = lane * V; k < g.K; k += 64 * V) {
                    const mtk_vec<T> a = k + V <= g.K ? mtk_ld(ap + k) : mtk_ld_n(ap + k, g.K - k), b = k + V <= g.K ? mtk_ld(xp + k) : mtk_ld_n(xp + k, g.K - k);
#pragma unroll
                    for (int i = 0; i < V; ++i) v += (float)a.v[i] * (float)b.v[i];
                }
                for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
                v *= g.scales ? g.scales[e] : g.scale;
            }
            if (lane == 0) us[q] = v;
        }
    }
    Acc acc = {};
#pragma unroll
    for (int l = 0; l < 2; ++l)
#pragma unroll
        for (int s = 0; s < S; ++s) acc = mma(wa[l][s], xa[l][s], acc);
    for (int k0 = (wave + 2 * NW) * KB; k0 < g.K; k0 += 2 * NW * KB) {
#pragma unroll
        for (int l = 0; l < 2; ++l) {
            const int kl = k0 + l * NW * KB;
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const int k = kl + s * LANES * V, left = g.K - k - hh * V;
                if (kl + KB <= g.K) {
                    xa[l][s] = mtk_ld(xr + k);
                    wa[l][s] = mtk_ld(wr + k);
                } else {
                    xa[l][s] = mtk_ld_n(xr + k, left);
                    wa[l][s] = mtk_ld_n(wr + k, left);
                }
            }
        }
#pragma unroll
        for (int l = 0; l < 2; ++l)
#pragma unroll
            for (int s = 0; s < S; ++s) acc = mma(wa[l][s], xa[l][s], acc);
    }
    // D[feature][row]: lane -> row; 32: register -> feature (reg & 3) + 8 (reg >> 2) + 4 (lane >> 5), 16: 4 (lane >> 4) + reg
    if constexpr (TS == 32) {
#pragma unroll
        for (int q = 0; q < 16; ++q) part[wave][li][(q & 3) + 8 * (q >> 2) + 4 * hh] = acc[q];
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) part[wave][li][4 * hh + q] = acc[q];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < OUT; ++i) {
        const int64_t row = m0 + rr + 16 * i;
        if (rr + 16 * i >= TS || row >= g.M || n >= g.N) continue;
        float v = bv;
#pragma unroll
        for (int w = 0; w < NW; ++w) v += part[w][rr + 16 * i][tid & (TS - 1)];
        if (FUSED && who[i] >= 0) {
            const float* ui = us + row * g.r;
            const T* br = up + ((int64_t)who[i] * g.N + n) * g.r;
            float low = 0.f;
#pragma unroll
            for (int p = 0; p < LP; ++p)
#pragma unroll
                for (int c = 0; c < V; ++c)
                    if (p * V + c < g.r) low += ui[p * V + c] * (float)ba[i][p].v[c];
            for (int j = LP * V; j < g.r; ++j) low += ui[j] * (float)br[j];
            v += low;
        } else if (who[i] >= 0) {
            float low = 0.f;
#pragma unroll
            for (int p = 0; p < LP; ++p)
#pragma unroll
                for (int c = 0; c < V; ++c) low += value(ua[i][p], c) * (float)ba[i][p].v[c];
            const L* ur = u + row * g.rp;
            const T* br = up + ((int64_t)who[i] * g.N + n) * g.r;
            for (int j = LP * V; j < g.r; j += V) {
                mtk_vec<L> uv[H];
#pragma unroll
                for (int h = 0; h < H; ++h) uv[h] = mtk_ld(ur + h * sec + j);
                const mtk_vec<T> bq = j + V <= g.r ? mtk_ld(br + j) : mtk_ld_n(br + j, g.r - j);
#pragma unroll
                for (int c = 0; c < V; ++c) low += value(uv, c) * (float)bq.v[c];
            }
            v += low;
        }
        if (g.relu) v = v < 0.f ? 0.f : v;
        y[row * g.N + n] = (T)v;
    }
    if (FUSED && n0 == 0) {  // u for the backward, laid out as k_shrink does
        for (int i = tid; i < (int)g.M * g.rp; i += 512) {
            const int row = i / g.rp, at = i - row * g.rp, c = at / sec, j = at - c * sec;
            L n[H];
            parts_of(c < kSections<T> && j < g.r ? us[row * g.r + j] : 0.f, n);
            L o = n[0];
#pragma unroll
            for (int h = 1; h < H; ++h) o = section_part(c) == h ? n[h] : o;
            u_out[i] = o;
        }
        if (uT) {
            const int64_t plane = mtk_up(g.r, 64) * g.Mp;
            for (int i = tid; i < (int)(mtk_up(g.r, 16) * g.Mp); i += 512) {
                const int j = i / (int)g.Mp, row = i - j * (int)g.Mp;
                L n[H];
                parts_of(j < g.r && row < g.M ? us[row * g.r + j] : 0.f, n);
#pragma unroll
                for (int h = 0; h < H; ++h) uT[h * plane + i] = n[h];
            }
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
// (chunk, model) pair raises c, e or both, so c + e numbers the pairs without bookkeeping.  Bound by reading x: four waves share a strip
// of columns and take the chunk's row groups in turn, the next group's loads in flight under the current one's products; their sums
// meet in LDS.  Two such products (down's and up's gradient) share a launch.
// 16-bit types: MFMA 16 x 16 x 32, the rows are its k.  u^T gives a lane's eight rows of one j as one piece; x's eight rows of eight
// columns come as eight pieces and are turned in registers, with fp16 into two bf16 numbers (exact) as B_e is.  fp32: 16 x 16 x 4, a lane holds one row's four columns and one j.
// Rows of other models are zeroed in BOTH operands (0 x inf).  65,536 rows of 1,024 bf16, both factors: 59 us (268 MB: 4.6 TB/s); the join 7 us.
template <typename T> constexpr int kStrip = sizeof(T) == 4 ? 64 : 128;  // columns of a workgroup
template <typename T, int JT>
__device__ void wgrad_body(const WgradArgs& g, int strip, int c, int j0, const Low<T>* __restrict__ u, const Low<T>* __restrict__ uT, const T* __restrict__ x, float* __restrict__ part,
                           float (*sum)[64 * 4]) {
    constexpr int V = mtk_piece<T>::n, NV = V;  // columns per lane
    constexpr int GR = sizeof(T) == 4 ? 16 : 32, PL = sizeof(T) == 4 ? 4 : 8;  // rows of a group, pieces of x per lane
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, q = lane >> 4;
    // A lane's columns.  One that would pass the last takes the last NV (again) and stores its own; only a layer narrower than that has no such.
    const int own0 = strip * kStrip<T> + li * NV, c0 = own0 + NV <= g.D ? own0 : g.D - NV;
    const int64_t lo = (int64_t)c * g.chunk, hi = lo + g.chunk < g.M ? lo + g.chunk : g.M;
    Owners own(g.offsets, g.E, lo, hi);
    int e;
    int64_t a, b;
    const int jp = (int)mtk_up(g.r, kRankT);
    while (own.next(e, a, b)) {
        f32x4 acc[JT][NV] = {};
        mtk_vec<T> xv[PL];
        T us[sizeof(T) == 4 ? PL : 1][JT];
        constexpr int P = kParts<T>;
        mtk_vec<Low<T>> ut[P][JT];  // the numbers of u
        // A scalar base and one 32-bit offset per lane.  A group with rows of other models clamps its rows to this one's and clears what it read
        // for them: a load that is made under a condition costs a branch (2,048 rows of 16 models in bf16: 21 us with such loads, 12 without)
        const int64_t plane = mtk_up(g.r, 64) * g.Mp;
        const unsigned ld = (unsigned)g.x_ld * (unsigned)sizeof(T);
        const unsigned first_row = sizeof(T) == 4 ? q : q * 8;
        auto load = [&](int64_t r0) {
            const bool inside = r0 >= a && r0 + GR <= b;
            const int64_t base_row = r0 < a ? a : r0;
            const char* base = (const char*)(x + base_row * g.x_ld);
            const int lo_r = r0 < a ? (int)(a - r0) : 0, hi_r = b - r0 < GR ? (int)(b - r0) : GR;  // this model's rows of the group
            const int skip = (int)(base_row - r0);
            if (g.D >= NV && g.x_ld < (1 << 24)) {
#pragma unroll
                for (int i = 0; i < PL; ++i) {
                    int row = (int)first_row + (sizeof(T) == 4 ? 4 : 1) * i;
                    if (!inside) row = row < lo_r ? lo_r : row >= hi_r ? hi_r - 1 : row;
                    xv[i] = mtk_ld((const T*)(base + (unsigned)(row - skip) * ld + (unsigned)c0 * (unsigned)sizeof(T)));
                }
            } else {
                for (int i = 0; i < PL; ++i) {
                    const int row = (int)first_row + (sizeof(T) == 4 ? 4 : 1) * i, rc = row < lo_r ? lo_r : row >= hi_r ? hi_r - 1 : row;
                    const T* xp = x + (r0 + rc) * g.x_ld;
#pragma unroll
                    for (int k = 0; k < NV; ++k) xv[i].v[k] = c0 + k >= 0 && c0 + k < g.D ? xp[c0 + k] : T(0);
                }
            }
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int i = 0; i < PL; ++i) {
                    const int row = (int)first_row + 4 * i, rc = row < lo_r ? lo_r : row >= hi_r ? hi_r - 1 : row;
#pragma unroll
                    for (int t = 0; t < JT; ++t) {
                        const int j = j0 + t * 16 + li;
                        us[i][t] = u[(r0 + rc) * g.rp + (j < g.rp ? j : g.rp - 1)];  // (a row behind the rank: never stored)
                    }
                }
            } else {
#pragma unroll
                for (int t = 0; t < JT; ++t)
#pragma unroll
                    for (int h = 0; h < P; ++h) ut[h][t] = mtk_ld(uT + h * plane + (int64_t)(j0 + t * 16 + li) * g.Mp + r0 + q * 8);
            }
            if (!inside) {
                auto clear = [](auto& v, uint4 m) {
                    const uint4 w = __builtin_bit_cast(uint4, v);
                    v = __builtin_bit_cast(typename std::remove_reference<decltype(v)>::type, make_uint4(w.x & m.x, w.y & m.y, w.z & m.z, w.w & m.w));
                };
                auto keeps = [&](int row) { return row >= lo_r && row < hi_r ? 0xffffffffu : 0u; };
#pragma unroll
                for (int i = 0; i < PL; ++i) {
                    const unsigned k = keeps((int)first_row + (sizeof(T) == 4 ? 4 : 1) * i);
                    clear(xv[i], make_uint4(k, k, k, k));
                    if constexpr (sizeof(T) == 4)
#pragma unroll
                        for (int t = 0; t < JT; ++t) us[i][t] = k ? us[i][t] : 0.f;
                }
                if constexpr (sizeof(T) == 2) {
                    unsigned m[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) m[i] = (keeps((int)first_row + 2 * i) & 0xffffu) | (keeps((int)first_row + 2 * i + 1) & 0xffff0000u);
#pragma unroll
                    for (int t = 0; t < JT; ++t)
#pragma unroll
                        for (int h = 0; h < P; ++h) clear(ut[h][t], make_uint4(m[0], m[1], m[2], m[3]));
                }
            }
        };
        const int64_t start = a / GR * GR + wave * GR;
        if (start < b) load(start);
        for (int64_t r0 = start; r0 < b; r0 += 4 * GR) {
            mtk_vec<T> xc[PL];
            mtk_vec<Low<T>> uc[P][JT];
            T uu[sizeof(T) == 4 ? PL : 1][JT];
#pragma unroll
            for (int i = 0; i < PL; ++i) xc[i] = xv[i];
#pragma unroll
            for (int t = 0; t < JT; ++t) {
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int h = 0; h < P; ++h) uc[h][t] = ut[h][t];
                } else
#pragma unroll
                    for (int i = 0; i < PL; ++i) uu[i][t] = us[i][t];
            }
            if (r0 + 4 * GR < b) load(r0 + 4 * GR);
            if constexpr (kF16<T>) {
#pragma unroll
                for (int cc = 0; cc < NV; ++cc) {
                    mtk_vec<T> col;
                    mtk_vec<Low<T>> b, d;
#pragma unroll
                    for (int i = 0; i < 8; ++i) col.v[i] = xc[i].v[cc];
                    two_numbers(col, b, d);
#pragma unroll
                    for (int t = 0; t < JT; ++t) {  // small ones first
                        f32x4 a = mma16(uc[1][t], d, acc[t][cc]);
                        a = mma16(uc[0][t], d, mma16(uc[2][t], b, a));
                        acc[t][cc] = mma16(uc[0][t], b, mma16(uc[1][t], b, a));
                    }
                }
            } else if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int cc = 0; cc < NV; ++cc) {
                    mtk_vec<T> col;
#pragma unroll
                    for (int i = 0; i < 8; ++i) col.v[i] = xc[i].v[cc];
#pragma unroll
                    for (int t = 0; t < JT; ++t) acc[t][cc] = mma16(uc[0][t], col, mma16(uc[1][t], col, acc[t][cc]));
                }
            } else {
#pragma unroll
                for (int i = 0; i < PL; ++i)
#pragma unroll
                    for (int t = 0; t < JT; ++t)
#pragma unroll
                        for (int cc = 0; cc < NV; ++cc) acc[t][cc] = __builtin_amdgcn_mfma_f32_16x16x4f32(uu[i][t], xc[i].v[cc], acc[t][cc], 0, 0, 0);
            }
        }
        // D[j][column lane]: register i -> j = 4 (lane >> 4) + i, column li of set cc is c0 + cc.  Wave w adds up the registers with index w.
        float* o = part + (int64_t)(c + e) * jp * g.D;
#pragma unroll
        for (int t = 0; t < JT; ++t) {
#pragma unroll
            for (int h = 0; h < NV; h += 4) {  // four columns at a time through 16 KB
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<float4*>(&sum[wave * 4 + i][lane * 4]) = make_float4(acc[t][h][i], acc[t][h + 1][i], acc[t][h + 2][i], acc[t][h + 3][i]);
                __syncthreads();
                float4 v = *reinterpret_cast<float4*>(&sum[wave][lane * 4]);
#pragma unroll
                for (int w = 1; w < 4; ++w) {
                    const float4 p = *reinterpret_cast<float4*>(&sum[w * 4 + wave][lane * 4]);
                    v.x += p.x; v.y += p.y; v.z += p.z; v.w += p.w;
                }
                const int j = j0 + t * 16 + q * 4 + wave;
                const mtk_vec<float> ov = {{v.x, v.y, v.z, v.w}};
                float* op = o + (int64_t)j * g.D + c0 + h;
                if (j < g.r && own0 < g.D) {
                    if (c0 == own0) mtk_st(op, ov);
                    else
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (c0 + h + k >= own0) op[k] = ov.v[k];
                }
            }
        }
    }
}
template <typename T> struct WgradOne {
    WgradArgs g;
    int strips, chunks;
    const Low<T> *u, *uT;
    const T* x;
    float* part;
    T* out;
    int turn;
};
template <typename T> struct WgradBoth {
    WgradOne<T> p[2];
};
template <typename T, int JT>
__global__ __launch_bounds__(256) void k_wgrad(WgradBoth<T> both, int j0) {
    __shared__ float sum[16][64 * 4];
    const WgradOne<T>& p = both.p[blockIdx.y];
    // workgroups go round-robin over the 8 XCDs.  A chunk's strips share u and, more so, are run by one XCD: its L2 would be asked for one
    // 256-byte piece of every row otherwise, which is a few of its channels
    const unsigned idx = blockIdx.x >> 3;
    const int64_t c = (int64_t)(idx / (unsigned)p.strips) * 8 + (blockIdx.x & 7);
    if (c >= p.chunks) return;
    wgrad_body<T, JT>(p.g, (int)(idx % (unsigned)p.strips), (int)c, j0, p.u, p.uT, p.x, p.part, sum);
}

// out[e] = sum of model e's chunks in ascending order; [r][D], or [D][r] when `turn`.  A model without rows gets zeros.
template <typename T>
__global__ __launch_bounds__(256) void k_wgrad_join(WgradBoth<T> both) {
    const WgradOne<T>& p = both.p[blockIdx.z];
    const WgradArgs& g = p.g;
    if (!p.out) return;
    const int e = blockIdx.y;
    const int jp = (int)mtk_up(g.r, kRankT);
    const int64_t n = (int64_t)g.r * g.D, slice = (int64_t)jp * g.D;
    int64_t a = g.offsets[e], b = g.offsets[e + 1];
    a = a < 0 ? 0 : a;
    b = b < g.M ? b : g.M;
    const int64_t ca = a / g.chunk, cb = b > a ? (b - 1) / g.chunk : ca - 1;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t j = i / g.D, d = i - j * g.D;
        const float* s = p.part + (ca + e) * slice + i;
        float v = 0.f;
        int64_t c = ca;
        for (; c + 3 <= cb; c += 4, s += 4 * slice) {
            const float v0 = s[0], v1 = s[slice], v2 = s[2 * slice], v3 = s[3 * slice];
            v = ((v + v0) + v1) + v2 + v3;
        }
        for (; c <= cb; ++c, s += slice) v += *s;
        p.out[(int64_t)e * n + (p.turn ? d * g.r + j : i)] = (T)v;
    }
}

// ------------------------------------------------------------------------------------------------------------------ helpers
// k_prep: everything that has to be laid out before the products, in one launch.  A job owns consecutive workgroups.
enum { JOB_TURN, JOB_PAD, JOB_BIAS, JOB_OWNER, JOB_ODD, JOB_TURN_TWO, JOB_TWO };
struct Job {
    int type, first;      // first workgroup
    const void* src;
    void* dst;
    int64_t rows, ld;     // PAD: rows and source row stride; OWNER: rows of x; BIAS: padded length
    int R, C, ldo;        // TURN: [batch][R][C] -> [batch][C][ldo]; PAD: [rows][C] -> [rows][ldo]; zeros behind; BIAS: C values; OWNER: C tiles of R rows;
                          // ODD: four workgroups for each of the runs of `rows` values; TURN_TWO, TWO: as TURN and PAD, from fp16 to
                          // rows of sections of two bf16 numbers
    int E;                // OWNER
    int rep;              // TURN, PAD: a row repeats every rep elements (a multiple of 32)
};
constexpr int kJobs = 10;
struct Jobs {
    Job job[kJobs];
    int n = 0, blocks = 0;
    void add(Job j, int64_t nblocks) {
        j.first = blocks;
        blocks += (int)nblocks;
        job[n++] = j;
    }
};
constexpr int kPadPieces = 1024;  // 16-byte pieces of a PAD workgroup

template <typename T>
__device__ void prep_body(const Jobs& jobs, int block, float* lds) {
    constexpr int V = mtk_piece<T>::n;
    T (*tile)[33] = reinterpret_cast<T (*)[33]>(lds);
    int q = 0;
    while (q + 1 < jobs.n && block >= jobs.job[q + 1].first) ++q;
    const Job& j = jobs.job[q];
    const int64_t blk = block - j.first;
    if (j.type == JOB_TURN) {
        const int nc = (j.C + 31) / 32, nr = (j.ldo + 31) / 32;
        const int64_t bat = blk / (nc * nr);
        const int rest = (int)(blk - bat * nc * nr), c0 = rest % nc * 32, r0 = rest / nc * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
        const T* in = (const T*)j.src + bat * j.R * j.C;
        T* out = (T*)j.dst + bat * j.C * j.ldo;
        const int rs = r0 % j.rep;
        for (int i = ty; i < 32; i += 8) tile[i][tx] = rs + i < j.R && c0 + tx < j.C ? in[(int64_t)(rs + i) * j.C + c0 + tx] : T(0);
        __syncthreads();
        for (int i = ty; i < 32; i += 8)
            if (c0 + i < j.C && r0 + tx < j.ldo) out[(int64_t)(c0 + i) * j.ldo + r0 + tx] = tile[tx][i];
    } else if (kF16<T> && j.type == JOB_TURN_TWO) {
        if constexpr (kF16<T>) {
            const int nc = (j.C + 31) / 32, nr = (j.R + 31) / 32, sec = section<T>(j.R);
            const int64_t bat = blk / (nc * nr);
            const int rest = (int)(blk - bat * nc * nr), c0 = rest % nc * 32, r0 = rest / nc * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
            const T* in = (const T*)j.src + bat * j.R * j.C;
            Low<T>* out = (Low<T>*)j.dst + bat * j.C * j.ldo;
            for (int i = ty; i < 32; i += 8) tile[i][tx] = r0 + i < j.R && c0 + tx < j.C ? in[(int64_t)(r0 + i) * j.C + c0 + tx] : T(0);
            __syncthreads();
            for (int i = ty; i < 32; i += 8) {
                if (c0 + i >= j.C) break;
                Low<T>* row = out + (int64_t)(c0 + i) * j.ldo;
                Low<T> n[2];
                parts_of((float)tile[tx][i], n);
                if (r0 + tx < sec)
#pragma unroll
                    for (int c = 0; c < kSections<T>; ++c) row[c * sec + r0 + tx] = n[section_second(c)];
                if (r0 == 0)
                    for (int k = kSections<T> * sec + tx; k < j.ldo; k += 32) row[k] = Low<T>(0.f);
            }
        }
    } else if (kF16<T> && j.type == JOB_TWO) {  // four values a thread
        if constexpr (kF16<T>) {
            struct __attribute__((aligned(8), may_alias)) Quad { Low<T> v[4]; };
            const int sec = section<T>(j.C), quads = sec / 4;
            const int64_t p = blk * 256 + threadIdx.x, at = p / quads;
            if (at < j.rows) {
                const int k0 = (int)(p - at * quads) * 4;
                const T* in = (const T*)j.src + at * j.ld + k0;
                Low<T>* row = (Low<T>*)j.dst + at * j.ldo;
                Quad o[2];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    Low<T> n[2];
                    parts_of(k0 + i < j.C ? (float)in[i] : 0.f, n);
                    o[0].v[i] = n[0];
                    o[1].v[i] = n[1];
                }
#pragma unroll
                for (int c = 0; c < kSections<T>; ++c) *reinterpret_cast<Quad*>(row + c * sec + k0) = o[section_second(c)];
                for (int k = kSections<T> * sec + k0; k < j.ldo; k += sec) *reinterpret_cast<Quad*>(row + k) = Quad{};
            }
        }
    } else if (j.type == JOB_PAD) {  // ldo is a multiple of a piece, dst 16-byte aligned
        const int ppr = j.ldo / V;
        const int64_t n = j.rows * ppr;
        for (int64_t p = blk * kPadPieces + threadIdx.x; p < n && p < (blk + 1) * kPadPieces; p += 256) {
            const int64_t row = p / ppr;
            const int c = (int)(p - row * ppr) * V % j.rep;
            const T* in = (const T*)j.src + row * j.ld + c;
            const mtk_vec<T> v = c + V <= j.C ? mtk_ld(in) : mtk_ld_n(in, j.C - c);
            *reinterpret_cast<uint4*>((T*)j.dst + p * V) = __builtin_bit_cast(uint4, v);
        }
    } else if (j.type == JOB_BIAS) {
        const int64_t i = blk * 256 + threadIdx.x;
        if (i < j.rows) ((float*)j.dst)[i] = i < j.C ? (float)((const T*)j.src)[i] : 0.f;
    } else if (j.type == JOB_OWNER) {
        const int64_t i = blk * 4 + (threadIdx.x >> 6);  // a wave a tile
        if (i < j.C) {
            const Owners own((const int32_t*)j.src, j.E, 0, 0);
            const TileModels m = TileModels::of_tile(own, i * j.R, j.R, j.rows, j.E);
            if ((threadIdx.x & 63) == 0) ((int32_t*)j.dst)[i] = m.packed();
        }
    } else {  // ODD: a byte each, so nobody clears them first
        const int64_t run = blk >> 2, share = blk & 3, pieces = (j.rows + V - 1) / V;
        const T* in = (const T*)j.src + run * j.rows;
        bool odd = false;
        for (int64_t p = share * 256 + threadIdx.x; p < pieces; p += 1024) {
            const int64_t left = j.rows - p * V;
            const mtk_vec<T> v = left >= V ? mtk_ld(in + p * V) : mtk_ld_n(in + p * V, (int)left);
#pragma unroll
            for (int i = 0; i < V; ++i) odd |= !(fabsf((float)v.v[i]) <= 3.4028235e38f);
        }
        odd = __syncthreads_or(odd);
        if (threadIdx.x == 0) ((unsigned char*)j.dst)[blk] = odd;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_prep(Jobs jobs) {
    __shared__ float lds[32 * 33];
    prep_body<T>(jobs, (int)blockIdx.x, lds);
}
// the shrink and what neither waits for the other: the jobs' workgroups run under its own (behind them: in front they leave the CUs' free
// places uneven: 65,536 rows of 64 models in bf16 56 us for 39)
template <typename T, int RT, int KS>
__global__ __launch_bounds__(256) void k_shrink(ShrinkArgs g, Jobs jobs, int j0, const T* __restrict__ x, const T* __restrict__ F, Low<T>* __restrict__ u, Low<T>* __restrict__ uT) {
    __shared__ float lds[kShrinkLds<RT, KS> > 32 * 33 ? kShrinkLds<RT, KS> : 32 * 33];
    const int own = g.tiles * g.turns;
    if ((int)blockIdx.x < own) shrink_body<T, RT, KS>(g, blockIdx.x, j0, x, F, u, uT, lds);
    else prep_body<T>(jobs, (int)blockIdx.x - own, lds);
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

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Rows of a chunk.  Both products' workgroups fill the CUs once (two of a CU fit with 16-bit rows, four with fp32): 65,536 rows of 1,024 in bf16
// 60 us, with three times as many 73 us.  An odd multiple of 64: chunks a power of two of bytes apart meet in the same memory channels (67 us).
int wgrad_chunk(int64_t M, int D, int dtype) {
    const int strip = dtype == MTK_DT_F32 ? 64 : 128, fill = dtype == MTK_DT_F32 ? 512 : 256;
    const int64_t c = cdiv(M * cdiv(D, strip), fill * 64);
    return (int)((c > 64 ? 64 : c) | 1) * 64;
}
int64_t wgrad_part(int64_t M, int D, int r, int E, int dtype) { return (cdiv(M, wgrad_chunk(M, D, dtype)) + E) * mtk_up(r, kRankT) * D; }

template <typename T, int RT>
void shrink_launch(ShrinkArgs g, const Jobs& jobs, int j0, const T* x, const T* F, Low<T>* u, Low<T>* uT, hipStream_t s) {
    // 32 rows a wave fill the chip from some 16,384 rows on; below, four waves split 16 rows
    const int turns = g.M >= 4096 ? 2 : g.M >= 2048 ? 4 : 16;
    g.turns = g.E < turns ? g.E : turns;
    g.tiles = (int)cdiv(g.M, g.M >= 16384 ? 128 : 16);
    const unsigned grid = (unsigned)(g.tiles * g.turns + jobs.blocks);
    if (g.M >= 16384) k_shrink<T, RT, 1><<<grid, 256, 0, s>>>(g, jobs, j0, x, F, u, uT);
    else k_shrink<T, RT, 4><<<grid, 256, 0, s>>>(g, jobs, j0, x, F, u, uT);
}
template <typename T>
void shrink(const ShrinkArgs& g, Jobs jobs, const T* x, const T* F, Low<T>* u, Low<T>* uT, hipStream_t s) {
    for (int j0 = 0; j0 < g.r; j0 += 64, jobs.n = jobs.blocks = 0) {
        if (g.r - j0 > 32) shrink_launch<T, 4>(g, jobs, j0, x, F, u, uT, s);
        else if (g.r - j0 > 16) shrink_launch<T, 2>(g, jobs, j0, x, F, u, uT, s);
        else shrink_launch<T, 1>(g, jobs, j0, x, F, u, uT, s);
    }
}
template <typename T>
WgradOne<T> wgrad_one(int64_t M, int64_t x_ld, int64_t Mp, int D, int r, int rp, int E, const int32_t* offsets, int dtype, int turn, const Low<T>* u, const Low<T>* uT, const T* x,
                      float* part, T* out) {
    const int chunk = wgrad_chunk(M, D, dtype);
    return WgradOne<T>{WgradArgs{M, x_ld, Mp, D, r, rp, E, chunk, offsets}, (int)cdiv(D, kStrip<T>), out ? (int)cdiv(M, chunk) : 0, u, uT, x, part, out, turn};
}
template <typename T>
void wgrad(const WgradBoth<T>& w, hipStream_t s) {
    const WgradOne<T>&p = w.p[0], &q = w.p[1];
    const int64_t n = (int64_t)p.strips * mtk_up(p.chunks, 8), m = (int64_t)q.strips * mtk_up(q.chunks, 8);
    const dim3 grid((unsigned)(n > m ? n : m), 2);
    for (int j0 = 0; j0 < p.g.r; j0 += 64) {
        if (p.g.r - j0 > 32) k_wgrad<T, 4><<<grid, 256, 0, s>>>(w, j0);
        else if (p.g.r - j0 > 16) k_wgrad<T, 2><<<grid, 256, 0, s>>>(w, j0);
        else k_wgrad<T, 1><<<grid, 256, 0, s>>>(w, j0);
    }
    const int64_t e = (int64_t)p.g.r * (p.g.D > q.g.D ? p.g.D : q.g.D);
    k_wgrad_join<T><<<dim3((unsigned)(cdiv(e, 256) < 1024 ? cdiv(e, 256) : 1024), p.g.E, 2), 256, 0, s>>>(w);
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
        u = l.take(M * rank_pad(r, dtype) * mtk_dtype_size(dtype));
        uT = dtype == MTK_DT_F32 ? l.at : l.take((dtype == MTK_DT_F16 ? kParts<mtk_f16> : kParts<mtk_bf16>) * Mp * mtk_up(r, 64) * mtk_dtype_size(dtype));
        bytes = l.at;
    }
};

// How a product [M x K] [N x K]^T runs.  few: k_linear_few; else a tile of k_linear.
struct Shape {
    bool few, blocks;  // blocks: the low-rank product as k-blocks (a model owns a tile's rows on average)
    int kind, BM, BN;  // 0: 256 x 256, 1: 128 x 128, 2: 64 x 64
    int line, rp, low_ld, Kp;  // elements of a line; u's row; a row of B_e for the epilogue, in whole 16-byte pieces; K in whole lines
    int64_t MT;
    int nb_n;
    Shape(int64_t M, int N, int K, int r, int E, int dtype) {
        line = 128 / mtk_dtype_size(dtype);
        rp = rank_pad(r, dtype);
        low_ld = (int)mtk_up(r, 16 / mtk_dtype_size(dtype));
        Kp = (int)mtk_up(K, line);
        // few: up to 64 rows, and while its 32 x 32 tiles fit the 256 CUs once.  us for K = N = 1024 and 16 models, few / 64 x 64 tiles: bf16
        // 64 rows 7.1 / 17, 256 rows 12 / 13, 384 rows 21 / 13, 1,024 rows 42 / 12; fp32 256 rows 19 / 32, 384 rows 33 / 30, 1,024 rows 69 / 31
        few = M <= 64 || (M <= 512 && cdiv(M, 32) * cdiv(N, 32) <= 256);
        // 256 x 256 tiles (one workgroup a CU) where they fill their rounds over the CUs to four fifths; 64 x 64 while the chip is not full.  us for
        // K = N = 1024, 256 / 128 / 64: bf16 65,536 rows 145 / 193 / 261, 20,011 rows 67 / 56 / 81, 8,192 rows 36 / 28 / 36, 2,048 rows
        // 31 / 19 / 15; fp32 20,011 rows - / 355 / 378, 8,192 rows - / 157 / 162, 2,048 rows - / 80 / 48
        const int64_t t256 = cdiv(M, 256) * cdiv(N, 256), t128 = cdiv(M, 128) * cdiv(N, 128);
        if (dtype == MTK_DT_F32) kind = t128 >= 1024 ? 1 : 2;
        else kind = t256 * 5 >= cdiv(t256, 256) * 256 * 4 ? 0 : t128 > 256 ? 1 : 2;
        BM = BN = kind == 0 ? 256 : kind == 1 ? 128 : 64;
        blocks = M >= (int64_t)E * BM;
        // k_linear with RAW: in 256 x 256 tiles its accumulators spill.  us, 128 / 256: 65,536 rows of 512 models 241 / 291, of 1,000 296 / 413
        if (dtype == MTK_DT_F16 && !blocks && kind == 0) kind = 1, BM = BN = 128;
        MT = cdiv(M, BM);
        nb_n = (int)cdiv(N, BN);
    }
};
// what k_linear reads beside its operands, and their padded copies where they need one
struct Packed {
    int64_t X, W, F, Bp, bias, owner, odd, pairs;  // F: the factors that the shrink multiplies, in whole lines like X
    Packed(Layout& l, const Shape& sh, int64_t M, int N, int r, int E, int dtype, bool pad_x, bool pad_w, bool pad_low) {
        const int64_t z = mtk_dtype_size(dtype);
        X = l.take(!sh.few && pad_x ? M * sh.Kp * z : 0);
        W = l.take(!sh.few && pad_w ? (int64_t)N * sh.Kp * z : 0);
        F = l.take(!sh.few && pad_x ? (int64_t)E * r * sh.Kp * z : 0);
        Bp = l.take(sh.blocks ? (int64_t)E * N * sh.rp * z : pad_low ? (int64_t)E * N * sh.low_ld * z : 0);
        bias = l.take((int64_t)sh.nb_n * sh.BN * 4);
        owner = l.take(sh.blocks ? sh.MT * 4 : 0);
        odd = l.take(sh.blocks ? (int64_t)E * 4 : 0);
        pairs = l.take(sh.blocks ? (sh.MT + E) * sh.BM * sh.rp * z : 0);
    }
};
// rows that LDS-DMA can stream as they are: whole lines, 16-byte aligned, offsets inside a tile in 32 bits
bool streams(const void* p, int64_t ld, int K, int dtype) {
    const int64_t z = mtk_dtype_size(dtype);
    return (uintptr_t)p % 16 == 0 && ld * z % 16 == 0 && K % (128 / z) == 0 && ld * z < (1 << 22);
}
struct ForwardWork {
    int64_t bytes;
    Shape sh;
    Packed pk;
    ForwardWork(Layout l, int64_t M, int din, int dout, int r, int E, int dtype, bool pad_x, bool pad_w)
        : sh(M, dout, din, r, E, dtype), pk(l, sh, M, dout, r, E, dtype, pad_x, pad_w, !sh.few && r != sh.low_ld) {
        bytes = sh.few ? 0 : l.at;
    }
};
struct BackwardWork {
    int64_t Bt, Wt, At, t, g, part[2], bytes;
    Shape sh;
    Packed pk;
    BackwardWork(Layout l, int64_t M, int din, int dout, int r, int E, int dtype, bool relu, bool pad_g)
        : sh(M, din, dout, r, E, dtype), pk(l, sh, M, din, r, E, dtype, pad_g, true, false) {  // the weights are turned, so laid out anew
        const int64_t z = mtk_dtype_size(dtype);
        Bt = l.take((int64_t)E * r * sh.Kp * z);
        Wt = l.take(sh.few ? (int64_t)din * dout * z : 0);  // else pk.W
        At = l.take(sh.blocks && !sh.few ? 0 : (int64_t)E * sh.low_ld * din * z);
        t = l.take(Saved(M, r, dtype).bytes);
        g = l.take(relu ? M * dout * z : 0);
        part[0] = l.take(wgrad_part(M, din, r, E, dtype) * 4);
        part[1] = l.take(wgrad_part(M, dout, r, E, dtype) * 4);
        bytes = l.at;
    }
};

void job_turn(Jobs& jobs, const void* src, void* dst, int R, int C, int ldo, int batch, int rep = 1 << 30) {
    jobs.add(Job{JOB_TURN, 0, src, dst, 0, 0, R, C, ldo, 0, rep}, cdiv(C, 32) * cdiv(ldo, 32) * batch);
}
void job_pad(Jobs& jobs, const void* src, int64_t ld, void* dst, int64_t rows, int C, int ldo, int V, int rep = 1 << 30) {
    jobs.add(Job{JOB_PAD, 0, src, dst, rows, ld, 0, C, ldo, 0, rep}, cdiv(rows * (ldo / V), kPadPieces));
}
// the same for rows of sections
void job_turn_two(Jobs& jobs, const void* src, void* dst, int R, int C, int ldo, int batch) {
    jobs.add(Job{JOB_TURN_TWO, 0, src, dst, 0, 0, R, C, ldo, 0, 1}, cdiv(C, 32) * cdiv(R, 32) * batch);
}
void job_two(Jobs& jobs, const void* src, void* dst, int64_t rows, int C, int ldo) {
    jobs.add(Job{JOB_TWO, 0, src, dst, rows, C, 0, C, ldo, 0, 1}, cdiv(rows * (section<mtk_f16>(C) / 4), 256));
}
template <typename T> void prep(const Jobs& jobs, hipStream_t s) {
    if (jobs.blocks) k_prep<T><<<(unsigned)jobs.blocks, 256, 0, s>>>(jobs);
}

// CUs of the current device, and whether a kernel's LDS limit has been raised there
struct DeviceState {
    int cus = 0;
    bool lds[11] = {};
};
DeviceState* device_state() {
    static DeviceState st[64];
    int d = 0;
    if (hipGetDevice(&d) != hipSuccess || d < 0 || d >= 64) return nullptr;
    if (!st[d].cus) {
        int n = 0;
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, d) != hipSuccess || n < 8) return nullptr;
        st[d].cus = n;
    }
    return &st[d];
}

template <typename T, bool RAW, int WR, int WC, int MW, int NT, int DX, int DW>
int launch_linear(const LinearArgs& g, int which, hipStream_t s) {
    typedef Geo<WR, WC, MW, NT, DX, DW> G;
    DeviceState* st = device_state();
    if (!st) MTK_FAIL(MTK_ERR_HIP, "adapter product: no device properties");
    if (!st->lds[which]) {
        MTK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(k_linear<T, WR, WC, MW, NT, DX, DW, RAW>), hipFuncAttributeMaxDynamicSharedMemorySize, G::kLds));
        st->lds[which] = true;
    }
    const int64_t per_xcd = cdiv(g.MT * g.nb_n, 8), room = (int64_t)st->cus / 8 * G::kRoom;
    k_linear<T, WR, WC, MW, NT, DX, DW, RAW><<<(unsigned)(8 * (per_xcd < room ? per_xcd : room)), 64 * G::NW, G::kLds, s>>>(g);
    return MTK_OK;
}
template <typename T, bool RAW> int linear_tile(const Shape& sh, LinearArgs& g, hipStream_t s) {
    constexpr int base = RAW ? 8 : sizeof(T) == 4 ? 0 : std::is_same<T, mtk_bf16>::value ? 3 : 6;
    if constexpr (sizeof(T) == 2 && !RAW)
        if (sh.kind == 0) return launch_linear<T, RAW, 2, 4, 4, 2, 3, 2>(g, base, s);
    if (sh.kind == 1) return launch_linear<T, RAW, 4, 2, 1, 2, 3, 2>(g, base + 1, s);
    return launch_linear<T, RAW, 2, 2, 1, 1, 3, 2>(g, base + 2, s);
}
template <typename T> int linear(const Shape& sh, LinearArgs& g, T* y, hipStream_t s) {
    g.Y = y;
    if constexpr (kF16<T>)
        if (!sh.blocks) return linear_tile<T, true>(sh, g, s);
    return linear_tile<T, false>(sh, g, s);
}
template <typename T>
void linear_few(const FewArgs& g, const T* x, const T* W, const T* bias, const Low<T>* u, const T* up, T* y, hipStream_t s) {
    if (g.M <= 64) k_linear_few<T, 16, false><<<(unsigned)(cdiv(g.M, 16) * cdiv(g.N, 16)), 512, 0, s>>>(g, x, W, bias, u, up, y, nullptr, nullptr, nullptr);
    else k_linear_few<T, 32, false><<<(unsigned)(cdiv(g.M, 32) * cdiv(g.N, 32)), 512, 0, s>>>(g, x, W, bias, u, up, y, nullptr, nullptr, nullptr);
}
// the shrink and the product of a row or some
template <typename T>
void linear_fused(const FewArgs& g, const T* x, const T* W, const T* bias, const T* down, const T* up, Low<T>* u, Low<T>* uT, T* y, hipStream_t s) {
    k_linear_few<T, 16, true><<<(unsigned)cdiv(g.N, 16), 512, 0, s>>>(g, x, W, bias, u, up, y, down, u, uT);
}
// the jobs of a k_linear product: x and W padded where they do not stream, B_e in whole lines and a block of zeros, bias, tiles' models.
// `early`: what the shrink reads.  F: W [N][K], or its transpose [K][N] when `turned`; L: B [E][N][r], or [E][r][N]
template <typename T>
LinearArgs plan_linear(Jobs& early, Jobs& jobs, const Shape& sh, const Packed& pk, char* wb, int64_t M, int N, int K, int r, int E, int dtype, const T* x, int64_t x_ld,
                       const T* F, bool turned, const T* bias, const T* L, const Low<T>* u, const int32_t* offsets, int relu) {
    constexpr int V = mtk_piece<T>::n;
    LinearArgs g{};
    g.M = M; g.MT = sh.MT; g.N = N; g.nb_n = sh.nb_n;
    g.nkb = sh.Kp / sh.line; g.nkx = sh.blocks ? sh.rp / sh.line : 0;
    g.offsets = offsets; g.E = E; g.relu = relu; g.U = u; g.rp = sh.rp; g.r = r;
    g.X = x;
    g.x_ld = x_ld * sizeof(T);
    if (!streams(x, x_ld, K, dtype)) {
        job_pad(early, x, x_ld, wb + pk.X, M, K, sh.Kp, V);
        g.X = wb + pk.X;
        g.x_ld = sh.Kp * sizeof(T);
    }
    g.W = F;
    g.w_ld = sh.Kp * sizeof(T);
    if (turned) job_turn(jobs, F, wb + pk.W, K, N, sh.Kp, 1);
    else if (!streams(F, K, K, dtype)) job_pad(jobs, F, K, wb + pk.W, N, K, sh.Kp, V);
    if (turned || !streams(F, K, K, dtype)) g.W = wb + pk.W;
    g.bias = (const float*)(wb + pk.bias);
    const int64_t nbias = (int64_t)sh.nb_n * sh.BN;
    jobs.add(Job{JOB_BIAS, 0, bias, wb + pk.bias, nbias, 0, 0, bias ? N : 0, 0, 0, 1}, cdiv(nbias, 256));
    if (sh.blocks) {
        if (kF16<T> && turned) job_turn_two(jobs, L, wb + pk.Bp, r, N, sh.rp, E);
        else if (kF16<T>) job_two(jobs, L, wb + pk.Bp, (int64_t)E * N, r, sh.rp);
        else if (turned) job_turn(jobs, L, wb + pk.Bp, r, N, sh.rp, E, section<T>(r));
        else job_pad(jobs, L, r, wb + pk.Bp, (int64_t)E * N, r, sh.rp, V, section<T>(r));
        jobs.add(Job{JOB_ODD, 0, L, wb + pk.odd, (int64_t)N * r, 0, 0, 0, 0, E, 1}, (int64_t)E * 4);
        jobs.add(Job{JOB_OWNER, 0, offsets, wb + pk.owner, M, 0, sh.BM, (int)sh.MT, 0, E, 1}, cdiv(sh.MT, 4));
        g.owner = (const int32_t*)(wb + pk.owner);
        g.odd = (const int32_t*)(wb + pk.odd);
        g.pairs = wb + pk.pairs;
        g.Bp = g.low = wb + pk.Bp;
        g.low_ld = sh.rp;
    }
    return g;
}

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
extern "C" int mtk_adapter_streams(const void* p, int64_t ld, int K, int dtype) { return mtk_dtype_ok(dtype) && K > 0 && streams(p, ld, K, dtype); }
extern "C" int64_t mtk_adapter_work_bytes(int64_t M, int din, int dout, int r, int E, int dtype, int act, int backward, int rows_stream, int weight_streams) {
    if (M <= 0 || din <= 0 || dout <= 0 || r <= 0 || E <= 0 || !mtk_dtype_ok(dtype)) return 0;
    return backward ? BackwardWork(Layout(), M, din, dout, r, E, dtype, act == 1, !rows_stream).bytes
                    : ForwardWork(Layout(), M, din, dout, r, E, dtype, !rows_stream, !weight_streams).bytes;
}

extern "C" int mtk_adapter_forward(int64_t M, int din, int dout, int r, int E, int dtype, const void* x, int64_t x_ld, const void* W, const void* bias,
                                   const void* down, const void* up, const int32_t* offsets, const float* scales, double scale, int act, int keep,
                                   void* y, void* saved, int64_t saved_bytes, void* work, int64_t work_bytes, mtk_stream stream) {
    if (const int rc = adapter_check("mtk_adapter_forward", M, din, dout, r, E, dtype, x_ld, act)) return rc;
    if (M == 0) return MTK_OK;
    if (!x || !W || !down || !up || !offsets || !y || !saved) MTK_FAIL(MTK_ERR_ARG, "mtk_adapter_forward: null pointer");
    if (((uintptr_t)saved | (uintptr_t)work) % 256) MTK_FAIL(MTK_ERR_ARG, "mtk_adapter_forward: saved and work have to lie on 256 bytes");
    const Saved sv(M, r, dtype);
    if (saved_bytes < sv.bytes) MTK_FAIL(MTK_ERR_ARG, "mtk_adapter_forward: a buffer of %lld bytes for the low-rank rows, %lld needed", (long long)saved_bytes, (long long)sv.bytes);
    const ForwardWork wk(Layout(), M, din, dout, r, E, dtype, !streams(x, x_ld, din, dtype), !streams(W, din, din, dtype));
    if (wk.bytes && (!work || work_bytes < wk.bytes)) MTK_FAIL(MTK_ERR_ARG, "mtk_adapter_forward: workspace of %lld bytes, %lld needed", (long long)work_bytes, (long long)wk.bytes);
    int rc = MTK_OK;
    mtk_by_type(dtype, [&](auto tag) {
        typedef decltype(tag) T;
        const hipStream_t s = (hipStream_t)stream;
        const Shape& sh = wk.sh;
        Low<T>* u = (Low<T>*)((char*)saved + sv.u);
        Low<T>* uT = keep && sizeof(T) == 2 ? (Low<T>*)((char*)saved + sv.uT) : nullptr;
        ShrinkArgs sa{M, din, r, sh.rp, E, x_ld, offsets, scales, (float)scale, sv.Mp, (char*)work + wk.pk.pairs, sh.blocks && !sh.few ? sh.BM : 0, 1, 1};
        if (sh.few) {
            const FewArgs fa{M, x_ld, dout, din, r, sh.rp, E, act, offsets, scales, (float)scale, sv.Mp};
            if (M * r <= kFusedPairs && M <= 16) {
                linear_fused<T>(fa, (const T*)x, (const T*)W, (const T*)bias, (const T*)down, (const T*)up, u, uT, (T*)y, s);
                return;
            }
            shrink<T>(sa, Jobs(), (const T*)x, (const T*)down, u, uT, s);
            linear_few<T>(fa, (const T*)x, (const T*)W, (const T*)bias, u, (const T*)up, (T*)y, s);
            return;
        }
        Jobs early, jobs;
        LinearArgs g = plan_linear<T>(early, jobs, sh, wk.pk, (char*)work, M, dout, din, r, E, dtype, (const T*)x, x_ld, (const T*)W, false, (const T*)bias, (const T*)up, u,
                                      offsets, act);
        if (!sh.blocks) {
            g.low = up;
            g.low_ld = sh.low_ld;
            if (r != sh.low_ld) {
                job_pad(jobs, up, r, (char*)work + wk.pk.Bp, (int64_t)E * dout, r, sh.low_ld, mtk_piece<T>::n);
                g.low = (char*)work + wk.pk.Bp;
            }
        }
        // x padded to whole lines: the shrink reads them too (20,011 rows of 517 in fp16: 11 us for the lines and 13 for the shrink; 33 for
        // both in one launch from rows as they are).
        const T *sx = (const T*)x, *sf = (const T*)down;
        if (g.X != x) {
            job_pad(early, down, din, (char*)work + wk.pk.F, (int64_t)E * r, din, sh.Kp, mtk_piece<T>::n);
            sx = (const T*)g.X;
            sf = (const T*)((char*)work + wk.pk.F);
            sa.K = sh.Kp;
            sa.x_ld = sh.Kp;
        }
        prep<T>(early, s);
        shrink<T>(sa, jobs, sx, sf, u, uT, s);
        rc = linear<T>(sh, g, (T*)y, s);
    });
    if (rc) return rc;
    MTK_HIP(hipGetLastError());
    return MTK_OK;
}

extern "C" int mtk_adapter_backward(int64_t M, int din, int dout, int r, int E, int dtype, const void* x, int64_t x_ld, const void* W, const void* down,
                                    const void* up, const int32_t* offsets, const float* scales, double scale, int act, const void* y, const void* dy,
                                    const void* saved, void* dx, void* ddown, void* dup, void* work, int64_t work_bytes, mtk_stream stream) {
    if (const int rc = adapter_check("mtk_adapter_backward", M, din, dout, r, E, dtype, x_ld, act)) return rc;
    if (M == 0) return MTK_OK;
    if (!x || !W || !down || !up || !offsets || !dy || !saved || !work || (act && !y)) MTK_FAIL(MTK_ERR_ARG, "mtk_adapter_backward: null pointer");
    if (((uintptr_t)saved | (uintptr_t)work) % 256) MTK_FAIL(MTK_ERR_ARG, "mtk_adapter_backward: saved and work have to lie on 256 bytes");
    const Saved sv(M, r, dtype);
    // (under an activation the masked gradient is a copy in the workspace, aligned)
    const BackwardWork wk(Layout(), M, din, dout, r, E, dtype, act == 1, act ? !streams(nullptr, dout, dout, dtype) : !streams(dy, dout, dout, dtype));
    if (work_bytes < wk.bytes) MTK_FAIL(MTK_ERR_ARG, "mtk_adapter_backward: workspace of %lld bytes, %lld needed", (long long)work_bytes, (long long)wk.bytes);
    int rc = MTK_OK;
    mtk_by_type(dtype, [&](auto tag) {
        typedef decltype(tag) T;
        const hipStream_t s = (hipStream_t)stream;
        const Shape& sh = wk.sh;
        char* wb = (char*)work;
        const Low<T> *u = (const Low<T>*)((const char*)saved + sv.u), *uT = (const Low<T>*)((const char*)saved + sv.uT);
        Low<T> *t = (Low<T>*)(wb + wk.t + sv.u), *tT = (Low<T>*)(wb + wk.t + sv.uT);
        const T* g = (const T*)dy;
        if (act) {
            T* gz = (T*)(wb + wk.g);
            const int64_t n = M * dout, nb = cdiv(n, 256 * mtk_piece<T>::n);
            k_relu_grad<T><<<(unsigned)(nb < 65536 ? nb : 65536), 256, 0, s>>>(n, (const T*)y, g, gz);
            g = gz;
        }
        Jobs early, jobs;
        LinearArgs lin{};
        const bool padded = dx && !sh.few && !streams(g, dout, dout, dtype);  // g in whole lines, for all that reads it from here on
        const int gk = padded ? sh.Kp : dout;
        const T* graw = g;
        if (padded) g = (const T*)(wb + wk.pk.X);
        if (dx || ddown) job_turn(early, up, wb + wk.Bt, dout, r, gk, E);
        if (dx) {
            if (sh.few) job_turn(jobs, W, wb + wk.Wt, dout, din, dout, 1);
            else lin = plan_linear<T>(early, jobs, sh, wk.pk, wb, M, din, dout, r, E, dtype, graw, dout, (const T*)W, true, nullptr, (const T*)down, t, offsets, 0);
            if (sh.few || !sh.blocks) {
                job_turn(jobs, down, wb + wk.At, r, din, sh.few ? r : sh.low_ld, E);
                lin.low = wb + wk.At;
                lin.low_ld = sh.low_ld;
            }
        }
        prep<T>(early, s);
        if (dx || ddown)
            shrink<T>(ShrinkArgs{M, gk, r, sh.rp, E, gk, offsets, scales, (float)scale, sv.Mp, wb + wk.pk.pairs, dx && sh.blocks && !sh.few ? sh.BM : 0, 1, 1},
                      jobs, g, (const T*)(wb + wk.Bt), t, ddown && sizeof(T) == 2 ? tT : nullptr, s);
        if (dx) {
            if (sh.few) linear_few<T>(FewArgs{M, dout, din, dout, r, sh.rp, E, 0, offsets, scales, (float)scale, sv.Mp}, g, (const T*)(wb + wk.Wt), nullptr, t, (const T*)(wb + wk.At), (T*)dx, s);
            else rc = linear<T>(sh, lin, (T*)dx, s);
        }
        if (ddown || dup)
            wgrad<T>(WgradBoth<T>{{wgrad_one<T>(M, x_ld, sv.Mp, din, r, sh.rp, E, offsets, dtype, 0, t, tT, (const T*)x, (float*)(wb + wk.part[0]), (T*)ddown),
                                   wgrad_one<T>(M, gk, sv.Mp, dout, r, sh.rp, E, offsets, dtype, 1, u, uT, g, (float*)(wb + wk.part[1]), (T*)dup)}}, s);
    });
    if (rc) return rc;
    MTK_HIP(hipGetLastError());
    return MTK_OK;
}
