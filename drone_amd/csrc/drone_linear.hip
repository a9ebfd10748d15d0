// drone_linear.hip — y = act(x W^T + b) + residual and its gradient, for the policy networks a device-resident learner runs
// between env steps. Three products:
//   forward  Y[m][n]  = sum_k X[m][k] W[n][k]      bias, activation, residual and act'(z) in the epilogue
//   input    DX[m][k] = sum_n DZ[m][n] W[n][k]     DZ = dy * act'(z)
//   weight   DW[n][k] = sum_m DZ[m][n] X[m][k]     split over m, partial sums joined in a fixed order; db rides along
// A policy's layers have many rows and few columns, so most of them are bound by memory, small ones by latency, and only wide
// ones by the matrix cores. The forms, chosen by size, type and alignment alone (measured on one MI355X; a large copy moves
// 5.1 TB/s there, a large product runs at 1 310 TFLOP/s bf16 and 153 f32):
//   linear_kernel           any size and alignment: tiles through registers into LDS, dz formed on the way
//   linear_few_kernel       few rows: one 32 x 32 tile a workgroup, the reduction dealt out to its waves
//   linear_resident_kernel  reductions of at most 1 KiB a row: weights in registers, rows streaming through LDS
//   linear_stream_kernel    whole 16-byte pieces: tiles straight from memory to LDS (wide layers, wide gradients)
//   linear_back_kernel      narrow layers: the whole gradient in one pass over the rows
// Odd widths take the streaming gradients too, on operands laid out in whole pieces (linear_dz_kernel, linear_pad_kernel).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "drone_policy.hpp"

#include "../../include/drone_vec.h"

namespace drone {
namespace {

constexpr int kPieces = 8;  // 16-byte pieces of the reduction axis a tile row holds: 64 16-bit or 32 f32 elements
constexpr int kJoinThreads = 256;
constexpr long long kJoinBlocks = 1 << 22;  // of the join at most: a launch of 2^32 threads or more runs only some of them, without an error

template <class T> __device__ __forceinline__ float to_f(T v) { return (float)v; }
template <class T> __device__ __forceinline__ float to_slope(typename Elem<T>::Slope v) { return (float)v * (1.f / Elem<T>::kSlopeScale); }

// ---- activation: value and slope in 32 bits, by the hardware's exp2 and rcp (1 ulp each). f32 tensors: tanh by its series
// near zero and erf from the math library. 16-bit tensors: the instructions count (the epilogue of a narrow layer is as long as
// its product): |tanh| = 1 - 2 / (1 + exp 2|z|), 2e-6 of itself off at most, and below 0.1 (where that would lose 1e-7 / z) two
// terms of the series; erfc by Abramowitz & Stegun 7.1.26 (|error| <= 1.5e-7; relative to gelu 5e-5 at z = -3, 5e-4 at -4,
// 4e-3 at -6, where it is 6e-9), whose exp(-z^2/2) is also what the slope needs. The forms are chosen so that infinities give
// the limits (no 0 * inf) and NaNs stay. ----
template <int ACT, bool PRECISE>
__device__ __forceinline__ float activate(float z, float& slope) {
    switch (ACT) {
        case DRONE_ACTIVATION_RELU:
            slope = z > 0.f ? 1.f : 0.f;
            return z > 0.f ? z : (z != z ? z : 0.f);
        case DRONE_ACTIVATION_TANH: {
            if (PRECISE) {
                const float x = 2.f * __builtin_amdgcn_rcpf(1.f + __expf(2.f * fabsf(z)));  // 1 - |tanh z|
                const float q = z * z;
                const float series = z * (1.f + q * (-0.33333334f + q * (0.13333334f + q * (-0.05396825f + q * 0.02186949f))));
                const bool small = q < 0.0625f;  // the series' next term is 1e-8 of z there
                slope = small ? 1.f - series * series : x * (2.f - x);
                return small ? series : copysignf(1.f - x, z);
            }
            const float r = __builtin_amdgcn_rcpf(1.f + __expf(2.f * fabsf(z))), q = z * z;  // r: (1 - |tanh z|) / 2
            slope = 4.f * r * (1.f - r);
            return q < 0.01f ? z * (1.f + q * (-0.33333334f + q * 0.13333334f)) : copysignf(1.f - 2.f * r, z);  // (next term: 5e-8 of z)
        }
        case DRONE_ACTIVATION_SILU: {
            const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z)), c = fminf(fmaxf(z, -90.f), 90.f);
            slope = s + c * (s * (1.f - s));
            return z < -90.f ? 0.f : z * s;
        }
        case DRONE_ACTIVATION_GELU: {  // max(z, 0) - |z| Q(|z|), Q(x) = 1/2 erfc(x / sqrt 2)
            const float e = __expf(-0.5f * z * z);
            float tail;
            if (PRECISE) {
                tail = 0.5f * erfcf(fabsf(z) * 0.70710678f);
            } else {
                const float t = __builtin_amdgcn_rcpf(1.f + 0.23164189f * fabsf(z));
                tail = e * (t * (0.127414796f + t * (-0.142248368f + t * (0.7107068705f + t * (-0.7265760135f + t * 0.5307027145f)))));
            }
            const float c = fminf(fmaxf(z, -30.f), 30.f);
            slope = (z < 0.f ? tail : 1.f - tail) + c * (e * 0.39894228f);
            return fmaxf(z, 0.f) - fminf(fabsf(z), 30.f) * tail;
        }
        default:
            slope = 1.f;
            return z;
    }
}

// ---- memory: N elements at any element-aligned address. The vector accesses of gfx950 take unaligned global addresses, so
// rows of 333 halves move in 16-byte pieces like rows of 336, and only a row's last piece goes element by element ----
template <class S, int N> struct Vec { S e[N]; };

template <class S, int N>
__device__ __forceinline__ Vec<S, N> load_n(const S* p, long long left) {
    Vec<S, N> v;
    if (left >= N) {
        __builtin_memcpy(&v, p, sizeof(v));
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) v.e[e] = (S)0.f;
#pragma unroll
        for (int e = 0; e < N; e++) if (e < left) v.e[e] = p[e];
    }
    return v;
}

template <class S, int N>
__device__ __forceinline__ void store_n(S* p, long long left, const float* f) {
    Vec<S, N> v;
#pragma unroll
    for (int e = 0; e < N; e++) v.e[e] = (S)f[e];
    if (left >= N) {
        __builtin_memcpy(p, &v, sizeof(v));
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) if (e < left) p[e] = v.e[e];
    }
}

// Elements at ... at + N - 1 of a row of `end` elements, zero past its end, without a branch (a branch around each load of a
// tile makes the loads wait for one another) and without touching what lies behind the row: the last N elements, shifted.
template <class S, int N>
__device__ __forceinline__ Vec<S, N> load_end(const S* row, long long at, long long end) {
    if constexpr (sizeof(S) * N > 16) {
        const auto lo = load_end<S, N / 2>(row, at, end), hi = load_end<S, N / 2>(row, at + N / 2, end);
        Vec<S, N> v;
#pragma unroll
        for (int e = 0; e < N / 2; e++) { v.e[e] = lo.e[e]; v.e[N / 2 + e] = hi.e[e]; }
        return v;
    } else {
        using Bits = std::conditional_t<sizeof(S) * N == 16, unsigned __int128, uint64_t>;
        using Pack = Vec<S, N>;
        Bits bits = 0;
        if (end >= N) {  // the same for the launch
            const long long from = at < end - N ? at : end - N, shift = at - from;
            __builtin_memcpy(&bits, row + from, sizeof(bits));
            bits = shift >= N ? 0 : bits >> (int)(shift * sizeof(S) * 8);
            return __builtin_bit_cast(Pack, bits);
        }
        Vec<S, N> v;
#pragma unroll
        for (int e = 0; e < N; e++) v.e[e] = at + e < end ? row[at + e] : (S)0.f;
        return v;
    }
}

// ---- tiles in LDS: [row][8 pieces of 16 B], piece p of row r at p ^ swz(r): eight neighbouring rows read the same piece
// from eight different bank groups, and the transposing loader's lanes (four rows apart) write to eight as well ----
__device__ __forceinline__ int swz(int r) { return (r ^ (r >> 3)) & 7; }

// The matrix instruction leaves a lane the result rows 8 a + 4 half + b (a, b = 0 ... 3) of its first operand. The features
// are that operand. f32: in their order, four neighbours are a 16-byte piece and the two halves of the wave hold neighbouring
// pieces. 16-bit types: feature 16 half + 4 a + b of every 32 is put into that row, so that a lane owns 16 neighbours, 32
// bytes of one output row (262144 x 256 x 256 bf16: 133 us; pieces of 8 interleaved between the halves: 148; f32 the other way
// round, 65536 x 64 x 64: 23 against 17 us).
template <class T> __device__ __forceinline__ int feature_of(int i) { return sizeof(T) == 4 ? i : (i & ~31) | ((i & 4) << 2) | ((i & 24) >> 1) | (i & 3); }
template <class T> __device__ __forceinline__ int row_of_feature(int f) { return sizeof(T) == 4 ? f : (f & ~31) | ((f & 16) >> 2) | ((f & 12) << 1) | (f & 3); }
// The lane's q-th piece of 32 features begins here (registers q kE ... of its sixteen).
template <class T> __device__ __forceinline__ int piece_feature(int q, int half) { return sizeof(T) == 4 ? (2 * q + half) * 4 : half * 16 + q * 8; }

// One operand as it lies in memory. CONTIG tiles: [row][reduction]; the others: [reduction][row]. With `slope` (a dense
// companion) the element is v * slope: the dz of the gradient, formed in 32 bits and rounded once for the matrix core. That
// rounding is a choice: the 16-bit matrix instructions take no finer operand, and dz as a sum of two 16-bit numbers would be
// twice the matrix work and twice the bytes of dz. It makes dx and dw of a 16-bit layer sqrt(2) times as far from 64 bits as
// their own rounding does (of their norm, bf16 0.24 % instead of 0.17, f16 0.029 instead of 0.021), and f16 dz below 6e-5 lose
// bits as any f16 gradient there does (scale the loss). db adds up the 32-bit values.
template <class T>
struct Operand {
    const T* p;
    long long ld;
    const typename Elem<T>::Slope* slope;
    long long slope_ld;
};

// Holds ROWS x 8 pieces of a [row][reduction] operand: thread t takes piece t % 8 of rows t / 8 + i THREADS / 8. Rows past
// the end repeat the last one (their results are not stored), the reduction past its end is zero.
template <class T, int ROWS, int THREADS, bool FEATURES>
struct ContigTile {
    static constexpr int kE = Elem<T>::kE, kN = ROWS * kPieces / THREADS;
    Vec<T, kE> reg[kN];
    static __device__ __forceinline__ int lds_row(int i) { return (threadIdx.x >> 3) + i * (THREADS / 8); }
    __device__ __forceinline__ void load(const Operand<T>& o, long long row0, long long rows, long long k0, long long kend) {
        if (k0 + kPieces * kE <= kend) some<true>(o, row0, rows, k0, kend); else some<false>(o, row0, rows, k0, kend);
    }
    // WHOLE: no piece of the tile crosses the end (the same for the workgroup)
    template <bool WHOLE>
    __device__ __forceinline__ void some(const Operand<T>& o, long long row0, long long rows, long long k0, long long kend) {
        const long long k = k0 + (threadIdx.x & 7) * kE;
#pragma unroll
        for (int i = 0; i < kN; i++) {
            long long r = row0 + (FEATURES ? feature_of<T>(lds_row(i)) : lds_row(i));
            r = r < rows ? r : rows - 1;
            reg[i] = WHOLE ? load_n<T, kE>(o.p + r * o.ld + k, kE) : load_end<T, kE>(o.p + r * o.ld, k, kend);
            if (o.slope) {
                using S = typename Elem<T>::Slope;
                const auto q = WHOLE ? load_n<S, kE>(o.slope + r * o.slope_ld + k, kE) : load_end<S, kE>(o.slope + r * o.slope_ld, k, kend);
#pragma unroll
                for (int e = 0; e < kE; e++) reg[i].e[e] = (T)(to_f(reg[i].e[e]) * to_slope<T>(q.e[e]));
            }
        }
    }
    __device__ __forceinline__ void store(u32x4* lds) const {
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int r = lds_row(i);
            lds[r * kPieces + ((threadIdx.x & 7) ^ swz(r))] = __builtin_bit_cast(u32x4, reg[i]);
        }
    }
};

// Holds the same tile from a [reduction][row] operand: a thread takes kE reduction steps x 4 rows (kE loads of 4 elements)
// and turns them in registers, so the LDS tile and the fragment reads are those of the contiguous form. A tile with fewer
// blocks than threads is the work of whole waves (the features' from the last wave down, so that two small tiles share out).
template <class T, int ROWS, int THREADS, bool FEATURES>
struct TransTile {
    static constexpr int kE = Elem<T>::kE, kBlocks = ROWS / 4 * kPieces, kN = (kBlocks + THREADS - 1) / THREADS;
    static_assert(kBlocks % THREADS == 0 || (kBlocks < THREADS && kBlocks % 64 == 0), "whole waves");
    Vec<T, 4> reg[kN][kE];
    static __device__ __forceinline__ int block_of(int i) { return FEATURES ? THREADS - 1 - (int)threadIdx.x + i * THREADS : (int)threadIdx.x + i * THREADS; }
    static __device__ __forceinline__ bool idle(int b) { return kBlocks < THREADS && b >= kBlocks; }
    // add: the 32-bit dz of this thread's four rows is added up over the reduction (the bias gradient)
    __device__ __forceinline__ void load(const Operand<T>& o, long long row0, long long rows, long long k0, long long kend, bool add, float (&sum)[kN][4]) {
        if (k0 + kPieces * kE <= kend && row0 + ROWS <= rows) some<true>(o, row0, rows, k0, kend, add, sum); else some<false>(o, row0, rows, k0, kend, add, sum);
    }
    template <bool WHOLE>
    __device__ __forceinline__ void some(const Operand<T>& o, long long row0, long long rows, long long k0, long long kend, bool add, float (&sum)[kN][4]) {
        using S = typename Elem<T>::Slope;
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int b = block_of(i);
            if (idle(b)) continue;
            const long long r = row0 + (b % (ROWS / 4)) * 4, k = k0 + b / (ROWS / 4) * kE;
#pragma unroll
            for (int e = 0; e < kE; e++) {
                const bool in = WHOLE || k + e < kend;
                const long long at = in ? k + e : kend - 1;  // steps past the end: the last one's values, put to zero below
                Vec<T, 4> v = WHOLE ? load_n<T, 4>(o.p + at * o.ld + r, 4) : load_end<T, 4>(o.p + at * o.ld, r, rows);
                float f[4];
#pragma unroll
                for (int j = 0; j < 4; j++) f[j] = to_f(v.e[j]);
                if (o.slope) {
                    const auto q = WHOLE ? load_n<S, 4>(o.slope + at * o.slope_ld + r, 4) : load_end<S, 4>(o.slope + at * o.slope_ld, r, rows);
#pragma unroll
                    for (int j = 0; j < 4; j++) { f[j] *= to_slope<T>(q.e[j]); v.e[j] = (T)f[j]; }
                }
                if (!WHOLE)
#pragma unroll
                    for (int j = 0; j < 4; j++) { f[j] = in ? f[j] : 0.f; v.e[j] = in ? v.e[j] : (T)0.f; }
                if (add)
#pragma unroll
                    for (int j = 0; j < 4; j++) sum[i][j] += f[j];
                reg[i][e] = v;
            }
        }
    }
    __device__ __forceinline__ void store(u32x4* lds) const {
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int b = block_of(i);
            if (idle(b)) continue;
            const int r = (b % (ROWS / 4)) * 4, c = b / (ROWS / 4), at = FEATURES ? row_of_feature<T>(r) : r;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                Vec<T, kE> v;
#pragma unroll
                for (int e = 0; e < kE; e++) v.e[e] = reg[i][e].e[j];
                lds[(at + j) * kPieces + (c ^ swz(at + j))] = __builtin_bit_cast(u32x4, v);
            }
        }
    }
};

// D += A B^T over one pair of 16-byte pieces per lane (the lane's half of the wave picks the piece, so a step spans 32 B of
// the reduction axis). The order of the reduction inside a step is the same for both operands, which is all the product needs.
[[maybe_unused]] __device__ __forceinline__ void mfma(f32x16& d, const u32x4& a, const u32x4& b, float) {
#pragma unroll
    for (int e = 0; e < 4; e++) d = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(b[e]), d, 0, 0, 0);
}
[[maybe_unused]] __device__ __forceinline__ void mfma(f32x16& d, const u32x4& a, const u32x4& b, __bf16) {
    d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), d, 0, 0, 0);
}
[[maybe_unused]] __device__ __forceinline__ void mfma(f32x16& d, const u32x4& a, const u32x4& b, _Float16) {
    d = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), d, 0, 0, 0);
}

enum Product { kForward, kInput, kWeight };

template <class T, int ROWS, int THREADS, bool CONTIG, bool FEATURES> struct TileOf { using type = ContigTile<T, ROWS, THREADS, FEATURES>; };
template <class T, int ROWS, int THREADS, bool FEATURES> struct TileOf<T, ROWS, THREADS, false, FEATURES> { using type = TransTile<T, ROWS, THREADS, FEATURES>; };

// A unit of work: one output tile of one part of the reduction. Units go to the XCDs in eight contiguous ranges (workgroups
// go round the XCDs), parts outermost, feature tiles innermost: workgroups that read the same rows share an L2.
struct Unit { long long part, tm; int tn; bool none; };
__device__ __forceinline__ Unit unit_of(long long tiles, int tiles_n, long long units) {
    const long long per = (units + 7) / 8, u = (long long)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
    Unit r;
    r.none = (long long)(blockIdx.x >> 3) >= per || u >= units;
    r.part = u / tiles;
    const long long tile = u - r.part * tiles;
    r.tm = tile / tiles_n;
    r.tn = (int)(tile - r.tm * tiles_n);
    return r;
}

// What a lane does with its results: 16 features (piece_feature) of row row0 + 32 m + lane % 32 for each (n, m). Everything the
// epilogue reads is asked for before the first value is used.
template <class T, int ACT, int TM, int TN, bool WHOLE>
__device__ __forceinline__ void write_forward(const LinearArgs& a, const f32x16 (&acc)[TN][TM], long long row0, long long feat0) {
    using Slope = typename Elem<T>::Slope;
    constexpr int kE = Elem<T>::kE, kQ = 16 / kE;
    const int half = (threadIdx.x >> 5) & 1, l32 = threadIdx.x & 31;
    u32x4 b[TN][kQ], res[TM][TN][kQ];  // as they come: unpacked where they are used
    using Piece = Vec<T, kE>;
    auto feat_of = [&](int n, int q) { return feat0 + n * 32 + piece_feature<T>(q, half); };
    auto left_of = [&](int n, int q) { return WHOLE ? (long long)kE : a.out - feat_of(n, q); };
#pragma unroll
    for (int n = 0; n < TN; n++)
#pragma unroll
        for (int q = 0; q < kQ; q++) {
            b[n][q] = u32x4{0, 0, 0, 0};
            if (a.b && left_of(n, q) > 0) b[n][q] = __builtin_bit_cast(u32x4, load_n<T, kE>((const T*)a.b + feat_of(n, q), left_of(n, q)));
        }
    if (a.res)
#pragma unroll
        for (int m = 0; m < TM; m++) {
            long long row = row0 + m * 32 + l32;
            row = row < a.rows ? row : a.rows - 1;
#pragma unroll
            for (int n = 0; n < TN; n++)
#pragma unroll
                for (int q = 0; q < kQ; q++)
                    if (left_of(n, q) > 0) res[m][n][q] = __builtin_bit_cast(u32x4, load_n<T, kE>((const T*)a.res + row * a.res_ld + feat_of(n, q), left_of(n, q)));
        }
#pragma unroll
    for (int m = 0; m < TM; m++) {
        const long long row = row0 + m * 32 + l32;
        if (row >= a.rows) continue;
#pragma unroll
        for (int n = 0; n < TN; n++)
#pragma unroll
            for (int q = 0; q < kQ; q++) {
                const long long feat = feat_of(n, q), left = left_of(n, q);
                if (left <= 0) continue;
                float v[kE], s[kE];
                const Piece bias = __builtin_bit_cast(Piece, b[n][q]);
#pragma unroll
                for (int j = 0; j < kE; j++) { v[j] = activate<ACT, sizeof(T) == 4>(acc[n][m][kE * q + j] + to_f(bias.e[j]), s[j]); s[j] *= Elem<T>::kSlopeScale; }
                if (a.slope) store_n<Slope, kE>((Slope*)a.slope + row * a.out + feat, left, s);
                if (a.res) {
                    const Piece r = __builtin_bit_cast(Piece, res[m][n][q]);
#pragma unroll
                    for (int j = 0; j < kE; j++) v[j] += to_f(r.e[j]);
                }
                store_n<T, kE>((T*)a.y + row * a.y_ld + feat, left, v);
            }
    }
}

template <class T, int ACT, int TM, int TN>
__device__ __forceinline__ void write_forward_any(const LinearArgs& a, const f32x16 (&acc)[TN][TM], long long row0, long long feat0, bool whole) {
    if (whole) write_forward<T, ACT, TM, TN, true>(a, acc, row0, feat0); else write_forward<T, ACT, TM, TN, false>(a, acc, row0, feat0);
}

template <class T, Product P, int TM, int TN>
__device__ __forceinline__ void write_results(const LinearArgs& a, const f32x16 (&acc)[TN][TM], long long row0, long long nrows, long long feat0, long long nfeat, bool whole, long long part) {
    constexpr int kE = Elem<T>::kE;
    if constexpr (P == kForward) {
        switch (a.act) {  // the same for the whole launch: one branch, not one per value
            case DRONE_ACTIVATION_RELU: write_forward_any<T, DRONE_ACTIVATION_RELU, TM, TN>(a, acc, row0, feat0, whole); break;
            case DRONE_ACTIVATION_TANH: write_forward_any<T, DRONE_ACTIVATION_TANH, TM, TN>(a, acc, row0, feat0, whole); break;
            case DRONE_ACTIVATION_SILU: write_forward_any<T, DRONE_ACTIVATION_SILU, TM, TN>(a, acc, row0, feat0, whole); break;
            case DRONE_ACTIVATION_GELU: write_forward_any<T, DRONE_ACTIVATION_GELU, TM, TN>(a, acc, row0, feat0, whole); break;
            default: write_forward_any<T, DRONE_ACTIVATION_NONE, TM, TN>(a, acc, row0, feat0, whole);
        }
    } else {
        const int half = (threadIdx.x >> 5) & 1, l32 = threadIdx.x & 31;
        auto write = [&](auto is_whole) {
            constexpr bool kWhole = decltype(is_whole)::value;  // no feature group crosses the end: no branch between the accesses
#pragma unroll
            for (int m = 0; m < TM; m++) {
                const long long row = row0 + m * 32 + l32;
                if (row >= nrows) continue;
#pragma unroll
                for (int n = 0; n < TN; n++)
#pragma unroll
                    for (int q = 0; q < 16 / kE; q++) {
                        const long long feat = feat0 + n * 32 + piece_feature<T>(q, half), left = kWhole ? kE : nfeat - feat;
                        if (left <= 0) continue;
                        float v[kE];
#pragma unroll
                        for (int j = 0; j < kE; j++) v[j] = acc[n][m][kE * q + j];
                        if (P == kInput) store_n<T, kE>((T*)a.dx + row * a.dx_ld + feat, left, v);
                        else store_n<float, kE>(a.work + part * a.out * a.in + row * a.in + feat, left, v);
                    }
            }
        };
        if (whole) write(std::true_type{}); else write(std::false_type{});
    }
}

// BM x BN outputs a workgroup (rows x features), WM x WN waves.
template <class T, Product P, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64, 2) void linear_kernel(LinearArgs a, float* db_work, int tiles_n, long long tiles, int parts, long long red_part) {
    using Slope = typename Elem<T>::Slope;
    constexpr int kThreads = WM * WN * 64, kE = Elem<T>::kE, kK = kPieces * kE, TM = BM / WM / 32, TN = BN / WN / 32;
    static_assert(TM >= 1 && TN >= 1 && BM % (kThreads / 8) == 0 && BN % (kThreads / 8) == 0, "a whole number of pieces for each thread");
    __shared__ u32x4 lds[2][(BM + BN) * kPieces];

    const Unit unit = unit_of(tiles, tiles_n, tiles * parts);
    if (unit.none) return;

    Operand<T> rowsop, featop;
    long long nrows, nfeat, red0 = 0, red1;
    const Slope* slope = (const Slope*)a.slope;
    if (P == kForward) {
        rowsop = {(const T*)a.x, a.x_ld, nullptr, 0};
        featop = {(const T*)a.w, a.w_ld, nullptr, 0};
        nrows = a.rows; nfeat = a.out; red1 = a.in;
    } else if (P == kInput) {
        rowsop = {(const T*)a.dy, a.dy_ld, slope, a.out};
        featop = {(const T*)a.w, a.w_ld, nullptr, 0};
        nrows = a.rows; nfeat = a.in; red1 = a.out;
    } else {
        rowsop = {(const T*)a.dy, a.dy_ld, slope, a.out};
        featop = {(const T*)a.x, a.x_ld, nullptr, 0};
        nrows = a.out; nfeat = a.in;
        red0 = unit.part * red_part;
        red1 = red0 + red_part < a.rows ? red0 + red_part : a.rows;
    }
    const long long row0 = unit.tm * BM, feat0 = (long long)unit.tn * BN;

    typename TileOf<T, BM, kThreads, P != kWeight, false>::type rt;
    typename TileOf<T, BN, kThreads, P == kForward, true>::type ft;
    constexpr int kSums = (BM / 4 * kPieces + kThreads - 1) / kThreads, kNoSums = (BN / 4 * kPieces + kThreads - 1) / kThreads;
    float sum[kSums][4] = {}, no_sum[kNoSums][4];
    const bool want_db = P == kWeight && a.db && unit.tn == 0;
    auto fetch = [&](long long k) {
        if constexpr (P == kWeight) rt.load(rowsop, row0, nrows, k, red1, want_db, sum); else rt.load(rowsop, row0, nrows, k, red1);
        if constexpr (P == kForward) ft.load(featop, feat0, nfeat, k, red1); else ft.load(featop, feat0, nfeat, k, red1, false, no_sum);
    };

    f32x16 acc[TN][TM] = {};
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, l32 = lane & 31;
    const int wrow = (wave / WN) * TM * 32, wfeat = (wave % WN) * TN * 32;

    if (red0 < red1) fetch(red0);
    int buf = 0;
    for (long long k = red0; k < red1; k += kK) {
        rt.store(lds[buf]);
        ft.store(lds[buf] + BM * kPieces);
        __syncthreads();
        if (k + kK < red1) fetch(k + kK);
        const u32x4* lr = lds[buf];
        const u32x4* lf = lds[buf] + BM * kPieces;
#pragma unroll
        for (int s = 0; s < kPieces / 2; s++) {
            u32x4 fr[TM], ff[TN];
#pragma unroll
            for (int i = 0; i < TM; i++) { const int r = wrow + i * 32 + l32; fr[i] = lr[r * kPieces + ((2 * s + half) ^ swz(r))]; }
#pragma unroll
            for (int i = 0; i < TN; i++) { const int r = wfeat + i * 32 + l32; ff[i] = lf[r * kPieces + ((2 * s + half) ^ swz(r))]; }
#pragma unroll
            for (int n = 0; n < TN; n++)
#pragma unroll
                for (int m = 0; m < TM; m++) mfma(acc[n][m], ff[n], fr[m], T{});
        }
        buf ^= 1;  // the next store goes to the other buffer; the barrier behind it says that everyone has left this one
    }

    write_results<T, P, TM, TN>(a, acc, row0 + wrow, nrows, feat0 + wfeat, nfeat, feat0 + BN <= nfeat, unit.part);
    if constexpr (P == kWeight) {
        if (want_db) {  // threads of one row group hold the sums of eight reduction pieces: joined in order through LDS
            float* join = (float*)lds;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kSums; i++) {
                const int b = threadIdx.x + i * kThreads;
                if (b < BM / 4 * kPieces)
#pragma unroll
                    for (int j = 0; j < 4; j++) join[(b / (BM / 4)) * BM + (b % (BM / 4)) * 4 + j] = sum[i][j];
            }
            __syncthreads();
            for (int i = threadIdx.x; i < BM && row0 + i < nrows; i += kThreads) {
                float s = 0.f;
#pragma unroll
                for (int c = 0; c < kPieces; c++) s += join[c * BM + i];
                db_work[unit.part * a.out + row0 + i] = s;
            }
        }
    }
}

// ---- the same three products with operands whose rows are whole, aligned 16-byte pieces (dz already formed): the tiles go
// from memory to LDS without passing through registers, one tile ahead of the matrix cores. A [reduction][row] operand
// keeps its order in LDS and is turned by the transposing LDS reads (16-bit types; f32 fragments are single values). ----
typedef short s16x4 __attribute__((ext_vector_type(4)));

// Natural tile of ROWS features: kE-element pieces, kP a row; the piece index is XORed by the reduction step so that the
// four (16-bit) or two (f32) steps one LDS access touches lie in different banks.
template <class T, int ROWS> struct NaturalSwz {
    static constexpr int kP = ROWS / Elem<T>::kE;
    static __device__ __forceinline__ int of(int m) { return sizeof(T) == 2 ? (kP >= 16 ? 4 * (m & 3) : 4 * ((m >> 1) & 1)) : kP >= 16 ? 8 * ((m >> 2) & 1) : 0; }
};

// PIECES 16-byte pieces of the reduction a row. Contiguous tiles: piece p of row r at p ^ piece_swz(r), so that the sixteen
// rows one LDS access takes lie in different banks.
template <int PIECES> __device__ __forceinline__ int piece_swz(int r) { return PIECES == 8 ? swz(r) : (r >> 2) & 3; }

template <class T, int ROWS, int PIECES, int WAVES, bool NATURAL, bool FEATURES>
struct StreamTile {
    static constexpr int kE = Elem<T>::kE, kP = ROWS / kE, kN = ROWS * PIECES / 64 / WAVES;
    static_assert(ROWS * PIECES % (64 * WAVES) == 0, "a whole number of loads for each wave");
    const T* base[kN];
    long long step;  // elements from one reduction step to the next
    __device__ __forceinline__ static int slot(int i) { return ((threadIdx.x >> 6) + i * WAVES) * 64 + (threadIdx.x & 63); }
    __device__ __forceinline__ static int offset(int i) {  // of the lane's piece, in reduction steps
        const int s = slot(i);
        return NATURAL ? s / kP : ((s % PIECES) ^ piece_swz<PIECES>(s / PIECES)) * kE;
    }
    __device__ __forceinline__ void init(const T* p, long long ld, long long row0, long long rows) {
        step = NATURAL ? ld : 1;
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int s = slot(i);
            if (NATURAL) {
                const int m = s / kP;
                long long f = row0 + ((s % kP) ^ NaturalSwz<T, ROWS>::of(m)) * kE;
                f = f < rows ? f : rows - kE;  // past the end: any piece of the row, its results are not stored
                base[i] = p + m * ld + f;
            } else {
                long long r = row0 + (FEATURES ? feature_of<T>(s / PIECES) : s / PIECES);
                r = r < rows ? r : rows - 1;
                base[i] = p + r * ld + offset(i);
            }
        }
    }
    // A whole tile from reduction step k on, straight into LDS: a wave's 64 lanes fill 1 KiB in order.
    __device__ __forceinline__ void stage(u32x4* lds, long long k) const {
#pragma unroll
        for (int i = 0; i < kN; i++)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(base[i] + k * step),
                                             (__attribute__((address_space(3))) void*)(lds + ((threadIdx.x >> 6) + i * WAVES) * 64), 16, 0, 0);
    }
    // The last, partial tile: zeros past the end of the reduction.
    __device__ __forceinline__ void stage_end(u32x4* lds, long long k, long long kend) const {
#pragma unroll
        for (int i = 0; i < kN; i++) {
            u32x4 v = {0, 0, 0, 0};
            if (k + offset(i) < kend) v = *(const u32x4*)(base[i] + k * step);
            lds[slot(i)] = v;
        }
    }
    // The lane's fragment of rows block ... block + 31 at step s (32 bytes of reduction).
    __device__ __forceinline__ static u32x4 fragment(const u32x4* lds, int block, int s) {
        const int lane = threadIdx.x & 63, half = lane >> 5, l32 = lane & 31;
        if constexpr (!NATURAL) {
            const int r = block + l32;
            return lds[r * PIECES + ((2 * s + half) ^ piece_swz<PIECES>(r))];
        } else if constexpr (sizeof(T) == 2) {
            // sixteen lanes turn a block of four steps x 16 features: lane j points at step j / 4, features 4 (j % 4) ...
            const int i = (lane & 16) + 4 * (lane & 3), f = block + (FEATURES ? feature_of<T>(i) : i), m0 = (lane & 15) >> 2;
            union { u32x4 u; s16x4 h[2]; } v;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int m = 16 * s + 8 * half + 4 * t + m0;
                const char* at = (const char*)(lds + m * kP + ((f / kE) ^ NaturalSwz<T, ROWS>::of(m))) + f % kE * 2;
                v.h[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
            }
            return v.u;
        } else {
            const int f = block + (FEATURES ? feature_of<T>(l32) : l32);
            u32x4 v;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int m = 8 * s + 4 * half + e;
                v[e] = ((const uint32_t*)(lds + m * kP + ((f / kE) ^ NaturalSwz<T, ROWS>::of(m))))[f % kE];
            }
            return v;
        }
    }
};

// Elements of a row of n with its last piece made whole (padded rows hold zeros there).
template <class T> __host__ __device__ __forceinline__ long long whole_pieces(long long n) { return (n + Elem<T>::kE - 1) / Elem<T>::kE * Elem<T>::kE; }

// Waits until at most LEFT of the wave's loads are under way (its LDS accesses all done), then for the workgroup.
template <int LEFT>
__device__ __forceinline__ void landed() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LEFT) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <class T, Product P, int BM, int BN, int WM, int WN, int PIECES, int STAGES>
__global__ __launch_bounds__(WM * WN * 64, 2) void linear_stream_kernel(LinearArgs a, int tiles_n, long long tiles, int parts, long long red_part) {
    constexpr int kE = Elem<T>::kE, kK = PIECES * kE, TM = BM / WM / 32, TN = BN / WN / 32;
    __shared__ u32x4 lds[STAGES][(BM + BN) * PIECES];
    const Unit unit = unit_of(tiles, tiles_n, tiles * parts);
    if (unit.none) return;
    long long nrows, nfeat, red0 = 0, red1;
    const long long row0 = unit.tm * BM, feat0 = (long long)unit.tn * BN;
    using RowTile = StreamTile<T, BM, PIECES, WM * WN, P == kWeight, false>;
    using FeatTile = StreamTile<T, BN, PIECES, WM * WN, P != kForward, true>;
    RowTile rt;
    FeatTile ft;
    if (P == kForward) {
        nrows = a.rows; nfeat = a.out; red1 = a.in;
        rt.init((const T*)a.x, a.x_ld, row0, nrows);
        ft.init((const T*)a.w, a.w_ld, feat0, nfeat);
    } else if (P == kInput) {
        nrows = a.rows; nfeat = a.in; red1 = a.out;
        rt.init((const T*)a.dy, a.dy_ld, row0, nrows);
        ft.init((const T*)a.w, a.w_ld, feat0, whole_pieces<T>(nfeat));
    } else {
        nrows = a.out; nfeat = a.in;
        red0 = unit.part * red_part;
        red1 = red0 + red_part < a.rows ? red0 + red_part : a.rows;
        rt.init((const T*)a.dy, a.dy_ld, row0, whole_pieces<T>(nrows));
        ft.init((const T*)a.x, a.x_ld, feat0, whole_pieces<T>(nfeat));
    }
    auto stage = [&](int to, long long k) {
        if (k + kK <= red1) {
            rt.stage(lds[to], k);
            ft.stage(lds[to] + BM * PIECES, k);
        } else if (k < red1) {
            rt.stage_end(lds[to], k, red1);
            ft.stage_end(lds[to] + BM * PIECES, k, red1);
        }
    };
    f32x16 acc[TN][TM] = {};
    const int wave = threadIdx.x >> 6, wrow = (wave / WN) * TM * 32, wfeat = (wave % WN) * TN * 32;
    // STAGES - 1 tiles under way. Tile i's loads are the oldest when its turn comes: the wait leaves the later tiles' out.
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) stage(i, red0 + (long long)i * kK);
    int buf = 0;
    for (long long k = red0; k < red1; k += kK) {
        if (k + (long long)(STAGES - 1) * kK <= red1) landed<(STAGES - 2) * (RowTile::kN + FeatTile::kN)>();
        else landed<0>();  // the last tiles: fewer, or one that went through registers, are behind this one
        const int next = buf == 0 ? STAGES - 1 : buf - 1;  // whose tile everyone has left at this barrier
        stage(next, k + (long long)(STAGES - 1) * kK);
        const u32x4* lr = lds[buf];
        const u32x4* lf = lds[buf] + BM * PIECES;
#pragma unroll
        for (int s = 0; s < PIECES / 2; s++) {
            u32x4 fr[TM], ff[TN];
#pragma unroll
            for (int i = 0; i < TM; i++) fr[i] = RowTile::fragment(lr, wrow + i * 32, s);
#pragma unroll
            for (int i = 0; i < TN; i++) ff[i] = FeatTile::fragment(lf, wfeat + i * 32, s);
#pragma unroll
            for (int n = 0; n < TN; n++)
#pragma unroll
                for (int m = 0; m < TM; m++) mfma(acc[n][m], ff[n], fr[m], T{});
        }
        buf = buf == STAGES - 1 ? 0 : buf + 1;
    }
    write_results<T, P, TM, TN>(a, acc, row0 + wrow, nrows, feat0 + wfeat, nfeat, feat0 + BN <= nfeat, unit.part);
}

// ---- a reduction of at most 1 KiB a row (512 16-bit, 256 f32): the weights stay in registers, 32 features a wave, and rows
// (with their residuals) stream through LDS. Persistent workgroups, all of LDS in row tiles under way, one barrier a tile:
// a tile costs its bytes and little else, where the tiled form pays a load latency for each of its few reduction steps and
// another for its epilogue. Loads into registers would spoil it: they retire in order behind the tiles under way, so the
// first one waits for them all (262144 x 256 x 256 bf16 with the residual in registers: 240 us). ----
constexpr int kResidentWaves = 8;

// Weight fragments of one wave: step s holds the lane's 16 bytes of feature lane % 32 from reduction 32-byte step s on.
template <class T, int KS>
__device__ __forceinline__ void load_weights(u32x4 (&w)[KS], const T* p, long long ld, int feat0, int nfeat, int red) {
    constexpr int kE = Elem<T>::kE;
    const int lane = threadIdx.x & 63, half = lane >> 5, f = feat0 + feature_of<T>(lane & 31);
#pragma unroll
    for (int s = 0; s < KS; s++) {
        const int k = (2 * s + half) * kE;
        w[s] = u32x4{0, 0, 0, 0};
        if (f < nfeat && k < red) w[s] = __builtin_bit_cast(u32x4, load_n<T, kE>(p + f * ld + k, red - k));
    }
}

// ROWS rows of PIECES 16-byte pieces in LDS, piece p of row r at p ^ swizzle(r) (sixteen rows' same piece in different banks).
template <class T, int ROWS, int PIECES>
struct RowTile {
    static constexpr int kE = Elem<T>::kE, kLoads = ROWS * PIECES / 64, kN = (kLoads + kResidentWaves - 1) / kResidentWaves;
    __device__ __forceinline__ static int swizzle(int r) { return PIECES >= 16 ? r & 15 : PIECES == 8 ? (r >> 1) & 7 : (r >> 2) & 3; }
    __device__ __forceinline__ static int at(int r, int piece) { return r * PIECES + (piece ^ swizzle(r)); }
    // The wave's i-th load: with fewer loads than waves some repeat another's, so that every wave has the same number under way.
    __device__ __forceinline__ static int load_of(int i) { return ((threadIdx.x >> 6) + i * kResidentWaves) % kLoads; }
    __device__ __forceinline__ static int slot(int i) { return load_of(i) * 64 + (threadIdx.x & 63); }
    __device__ __forceinline__ static int piece_of(int i) { return (slot(i) % PIECES) ^ swizzle(slot(i) / PIECES); }
    // Pieces past the row's end are never written: zero for good (a garbage x would make its product with a zero weight a NaN).
    __device__ __forceinline__ static void clear(u32x4* lds, int pieces) {
#pragma unroll
        for (int i = 0; i < kN; i++) if (piece_of(i) >= pieces) lds[slot(i)] = u32x4{0, 0, 0, 0};
    }
    // Every load covers at least one whole row, so none of a wave's loads is ever skipped (landed() counts them).
    static_assert(64 % PIECES == 0 || PIECES % 64 == 0, "whole rows");
    __device__ __forceinline__ static void stage(u32x4* lds, const T* p, long long ld, long long row0, long long rows, int pieces) {
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const long long r0 = row0 + slot(i) / PIECES, r = r0 < rows ? r0 : rows - 1;
            const int piece = piece_of(i);
            if (piece < pieces)
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(p + r * ld + piece * kE),
                                                 (__attribute__((address_space(3))) void*)(lds + load_of(i) * 64), 16, 0, 0);
        }
    }
};

template <class T, int KS, int WF, bool RES>
struct Resident {
    static constexpr int kE = Elem<T>::kE, kQ = 16 / kE, kRows = kResidentWaves / WF * 32;
    using X = RowTile<T, kRows, 2 * KS>;
    using R = RowTile<T, kRows, WF * 32 / kE>;
    static constexpr int kX = kRows * 2 * KS, kTile = kX + (RES ? kRows * WF * 32 / kE : 0);  // pieces
    // Tiles of LDS: two workgroups a CU where the registers allow it (short reductions), else one with most of the memory.
    static constexpr int kPerCu = KS <= 4 && kTile * 16 * 4 <= 72 * 1024 ? 2 : 1, kFit = 144 * 1024 / kPerCu / (kTile * 16), kStages = kFit > 8 ? 8 : kFit;
    static constexpr int kLoads = X::kN + (RES ? R::kN : 0);  // a wave's for one tile
    static_assert(kStages >= 2, "at least one tile ahead");
};

template <class T, int ACT, int KS, int WF, bool RES, bool SLOPE>
__device__ __forceinline__ void resident_forward(const LinearArgs& a, u32x4 (*lds)[Resident<T, KS, WF, RES>::kTile], int groups, int slots) {
    using M = Resident<T, KS, WF, RES>;
    using Slope = typename Elem<T>::Slope;
    constexpr int kE = M::kE, kQ = M::kQ, kBM = M::kRows, kStages = M::kStages;
    constexpr int kStores = kQ + (SLOPE ? kQ * kE * (int)sizeof(Slope) / 16 : 0);  // a wave's for one tile
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, r = (wave / WF) * 32 + (lane & 31);
    const int xcd = blockIdx.x & 7, at = blockIdx.x >> 3, group = at % groups, pieces = a.in / kE;
    const int tiles = (int)((a.rows + kBM - 1) / kBM), step = 8 * slots, group0 = group * WF * 32, feat0 = group0 + wave % WF * 32;
    int tile = xcd * slots + at / groups;
    if (tile >= tiles) return;
    auto stage = [&](int to, int t) {
        M::X::stage(lds[to], (const T*)a.x, a.x_ld, (long long)t * kBM, a.rows, pieces);
        if (RES) M::R::stage(lds[to] + M::kX, (const T*)a.res + group0, a.res_ld, (long long)t * kBM, a.rows, (a.out - group0) / kE);
    };
#pragma unroll
    for (int i = 0; i < kStages; i++) M::X::clear(lds[i], pieces);
    u32x4 w[KS], bias[kQ];
    load_weights<T, KS>(w, (const T*)a.w, a.w_ld, feat0, a.out, a.in);
    auto left = [&](int q) { return a.out - feat0 - piece_feature<T>(q, half); };
    auto column = [&](int q) { return feat0 + piece_feature<T>(q, half); };
#pragma unroll
    for (int q = 0; q < kQ; q++) {
        bias[q] = u32x4{0, 0, 0, 0};
        if (a.b && left(q) > 0) bias[q] = __builtin_bit_cast(u32x4, load_n<T, kE>((const T*)a.b + column(q), left(q)));
    }
#pragma unroll
    for (int i = 0; i < kStages - 1; i++)
        if (tile + i * step < tiles) stage(i, tile + i * step);
    const bool whole = feat0 + 32 <= a.out;  // the wave's stores all go out (its rows are whole up to the last tile)
    int buf = 0;
    for (int turn = 0; tile < tiles; tile += step, turn++) {
        // this tile's loads have kStages - 2 tiles' behind them, and from the kStages-th turn on as many tiles' stores and one more
        if (tile + (kStages - 2) * step >= tiles) landed<0>();
        else if (whole && turn >= kStages - 1) landed<((kStages - 2) * M::kLoads + (kStages - 1) * kStores < 63 ? (kStages - 2) * M::kLoads + (kStages - 1) * kStores : 63)>();
        else landed<(kStages - 2) * M::kLoads>();
        const int next = buf == 0 ? kStages - 1 : buf - 1;
        if (tile + (kStages - 1) * step < tiles) stage(next, tile + (kStages - 1) * step);
        f32x16 acc;
#pragma unroll
        for (int q = 0; q < kQ; q++) {
            const auto b = __builtin_bit_cast(Vec<T, kE>, bias[q]);
#pragma unroll
            for (int j = 0; j < kE; j++) acc[q * kE + j] = to_f(b.e[j]);
        }
#pragma unroll
        for (int s = 0; s < KS; s++) mfma(acc, w[s], lds[buf][M::X::at(r, 2 * s + half)], T{});
        const long long row = (long long)tile * kBM + r;
        auto write = [&](auto is_whole) {
#pragma unroll
            for (int q = 0; q < kQ; q++) {
                const int n = decltype(is_whole)::value ? kE : left(q);
                if (n <= 0) continue;
                float v[kE], s[kE];
#pragma unroll
                for (int j = 0; j < kE; j++) { v[j] = activate<ACT, sizeof(T) == 4>(acc[q * kE + j], s[j]); s[j] *= Elem<T>::kSlopeScale; }
                if (SLOPE) store_n<Slope, kE>((Slope*)a.slope + row * a.out + column(q), n, s);
                if (RES) {
                    const auto more = __builtin_bit_cast(Vec<T, kE>, lds[buf][M::kX + M::R::at(r, (column(q) - group0) / kE)]);
#pragma unroll
                    for (int j = 0; j < kE; j++) v[j] += to_f(more.e[j]);
                }
                store_n<T, kE>((T*)a.y + row * a.y_ld + column(q), n, v);
            }
        };
        if (row < a.rows) { if (whole) write(std::true_type{}); else write(std::false_type{}); }
        buf = buf == kStages - 1 ? 0 : buf + 1;
    }
}

template <class T, int KS, int WF, bool RES, int PER_CU>
__global__ __launch_bounds__(kResidentWaves * 64, 2 * PER_CU) void linear_resident_kernel(LinearArgs a, int groups, int slots) {
    __shared__ u32x4 lds[Resident<T, KS, WF, RES>::kStages][Resident<T, KS, WF, RES>::kTile];
    auto go = [&](auto act) {
        if (a.slope) resident_forward<T, decltype(act)::value, KS, WF, RES, true>(a, lds, groups, slots);
        else resident_forward<T, decltype(act)::value, KS, WF, RES, false>(a, lds, groups, slots);
    };
    switch (a.act) {
        case DRONE_ACTIVATION_RELU: go(std::integral_constant<int, DRONE_ACTIVATION_RELU>{}); break;
        case DRONE_ACTIVATION_TANH: go(std::integral_constant<int, DRONE_ACTIVATION_TANH>{}); break;
        case DRONE_ACTIVATION_SILU: go(std::integral_constant<int, DRONE_ACTIVATION_SILU>{}); break;
        case DRONE_ACTIVATION_GELU: go(std::integral_constant<int, DRONE_ACTIVATION_GELU>{}); break;
        default: go(std::integral_constant<int, DRONE_ACTIVATION_NONE>{});
    }
}

// dz = dy * slope, rounded once to T, into rows of whole pieces (or nowhere: dz is dy), and the bias gradient's partial
// sums of the 32-bit values: thread (c, g) of a workgroup owns piece c of a strip of kStrip pieces and every kGroups-th of the
// workgroup's rows.
template <class T, bool WHOLE>
__global__ __launch_bounds__(256) void linear_dz_kernel(LinearArgs a, T* dz, long long dz_ld, float* partial, long long rows_part) {
    using Slope = typename Elem<T>::Slope;
    constexpr int kE = Elem<T>::kE, kStrip = 32, kGroups = 8;
    __shared__ float join[kGroups][kStrip * kE];
    const int c = threadIdx.x % kStrip, g = threadIdx.x / kStrip;
    const long long col = ((long long)blockIdx.y * kStrip + c) * kE, left = a.out - col;
    const long long row0 = blockIdx.x * rows_part, row1 = row0 + rows_part < a.rows ? row0 + rows_part : a.rows;
    float sum[kE] = {};
    if (left > 0)
#pragma unroll 4
        for (long long r = row0 + g; r < row1; r += kGroups) {
            const auto v = WHOLE ? load_n<T, kE>((const T*)a.dy + r * a.dy_ld + col, kE) : load_end<T, kE>((const T*)a.dy + r * a.dy_ld, col, a.out);
            float f[kE];
#pragma unroll
            for (int e = 0; e < kE; e++) f[e] = to_f(v.e[e]);
            if (a.slope) {
                const auto q = WHOLE ? load_n<Slope, kE>((const Slope*)a.slope + r * a.out + col, kE) : load_end<Slope, kE>((const Slope*)a.slope + r * a.out, col, a.out);
#pragma unroll
                for (int e = 0; e < kE; e++) f[e] *= to_slope<T>(q.e[e]);
            }
            if (dz) store_n<T, kE>(dz + r * dz_ld + col, kE, f);
#pragma unroll
            for (int e = 0; e < kE; e++) sum[e] += f[e];
        }
    if (!partial) return;
#pragma unroll
    for (int e = 0; e < kE; e++) join[g][c * kE + e] = sum[e];
    __syncthreads();
    const long long first = (long long)blockIdx.y * kStrip * kE;
    for (int i = threadIdx.x; i < kStrip * kE && first + i < a.out; i += 256) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < kGroups; k++) s += join[k][i];
        partial[(long long)blockIdx.x * a.out + first + i] = s;
    }
}

// Rows of `cols` elements into rows of whole, aligned pieces, zeros behind their end.
template <class T>
__global__ __launch_bounds__(256) void linear_pad_kernel(const T* from, long long ld, long long rows, int cols, T* to, int pieces) {
    constexpr int kE = Elem<T>::kE;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows * pieces; i += (long long)gridDim.x * 256) {
        const long long r = i / pieces;
        const int p = (int)(i - r * pieces);
        *(u32x4*)(to + (r * pieces + p) * kE) = __builtin_bit_cast(u32x4, load_end<T, kE>(from + r * ld, p * kE, cols));
    }
}

// ---- the whole gradient of a narrow layer (up to 128 x 128, 256 x 64) in one pass: dy, the slopes and x are read
// once, dx is written once, the weight gradient stays in the accumulators of persistent workgroups until their last tile.
// A tile of rows arrives in LDS, is turned into dz there (each thread its own pieces, adding up the bias gradient), and is
// then the row operand of dx (weights in registers) and, read transposed, of the weight gradient. ----
constexpr int kBackThreads = 512, kBackWaves = 8;

// Piece p of row r at p ^ back_swz(r): sixteen rows' same piece in different banks (dx), and four neighbouring rows' 64-byte
// blocks too (the transposed reads).
template <int PIECES> __device__ __forceinline__ int back_swz(int r) {
    return PIECES >= 16 ? ((r & 3) << 2) | ((r >> 2) & 3) : PIECES == 8 ? ((r >> 1) & 1) << 2 | ((r >> 2) & 3) : (r >> 2) & 3;
}

// A [ROWS][PIECES] tile of LDS filled by eight waves; the same number of loads for every wave.
template <class E, int ROWS, int PIECES>
struct BackTile {
    static constexpr int kE = 16 / sizeof(E), kCount = ROWS * PIECES, kLoads = kCount / 64, kN = (kLoads + kBackWaves - 1) / kBackWaves;
    __device__ __forceinline__ static int at(int r, int piece) { return r * PIECES + (piece ^ back_swz<PIECES>(r)); }
    __device__ __forceinline__ static int load_of(int i) { return ((threadIdx.x >> 6) + i * kBackWaves) % kLoads; }
    __device__ __forceinline__ static int slot(int i) { return load_of(i) * 64 + (threadIdx.x & 63); }
    __device__ __forceinline__ static int row_of(int s) { return s / PIECES; }
    __device__ __forceinline__ static int piece_of(int s) { return (s % PIECES) ^ back_swz<PIECES>(s / PIECES); }
    __device__ __forceinline__ static void clear(u32x4* lds, int pieces) {
        for (int s = threadIdx.x; s < kCount; s += kBackThreads) if (piece_of(s) >= pieces) lds[s] = u32x4{0, 0, 0, 0};
    }
    __device__ __forceinline__ static void stage(u32x4* lds, const E* p, long long ld, long long row0, long long rows, int pieces) {
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int s = slot(i), piece = piece_of(s);
            const long long r0 = row0 + row_of(s), r = r0 < rows ? r0 : rows - 1;
            if (piece < pieces)  // (64 slots hold a whole row or more: some lane of every load takes part)
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(p + r * ld + piece * kE),
                                                 (__attribute__((address_space(3))) void*)(lds + load_of(i) * 64), 16, 0, 0);
        }
    }
    // Fragment of columns block ... block + 31 (as `features` of the product or as its rows) over the reduction step s of rows.
    template <bool FEATURES>
    __device__ __forceinline__ static u32x4 transposed(const u32x4* lds, int block, int row0) {
        const int lane = threadIdx.x & 63, half = lane >> 5;
        if constexpr (sizeof(E) == 2) {
            const int i = (lane & 16) + 4 * (lane & 3), f = block + (FEATURES ? feature_of<E>(i) : i), m0 = (lane & 15) >> 2;
            union { u32x4 u; s16x4 h[2]; } v;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int m = row0 + 8 * half + 4 * t + m0;
                v.h[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)((const char*)(lds + at(m, f / kE)) + f % kE * 2));
            }
            return v.u;
        } else {
            const int f = block + (lane & 31);
            u32x4 v;
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = ((const uint32_t*)(lds + at(row0 + 4 * half + e, f / kE)))[f % kE];
            return v;
        }
    }
};

template <class T, int OB, int IB>
struct Back {
    using Slope = typename Elem<T>::Slope;
    static constexpr int kE = Elem<T>::kE, kPo = OB * 32 / kE, kPi = IB * 32 / kE, kPs = OB * 32 / (16 / (int)sizeof(Slope));
    static constexpr int kRowBytes = (kPo + kPi + kPs) * 16;
    // rows of a tile: three tiles in LDS, at most 32 for each of the waves that share a feature block
    static constexpr int kMost = 32 * (kBackWaves / IB), kFit = 152 * 1024 / 3 / kRowBytes, kRows = kFit >= kMost ? kMost : kFit >= 128 ? (kMost < 128 ? kMost : 128) : kFit >= 64 ? (kMost < 64 ? kMost : 64) : 32;
    static constexpr int kTile = kRows * (kPo + kPi + kPs), kStages = 152 * 1024 / (kTile * 16) > 6 ? 6 : 152 * 1024 / (kTile * 16);
    static_assert(kStages >= 2 && kRows >= 32, "at least one tile ahead");
    using Dy = BackTile<T, kRows, kPo>;
    using X = BackTile<T, kRows, kPi>;
    using S = BackTile<Slope, kRows, kPs>;
    static constexpr int kS = kRows * kPo, kX = kS + kRows * kPs;  // offsets in a tile: dy, slopes, x
    static constexpr int kBlocks = OB * IB, kMine = kBlocks > kBackWaves ? kBlocks / kBackWaves : 1;      // 32 x 32 blocks of the weight gradient, a wave's
    static constexpr int kSlices = kBlocks < kBackWaves ? kBackWaves / kBlocks : 1;                       // waves that share a block, each its rows
    static constexpr int kStep = 32 / (int)sizeof(T);                                                     // rows of a reduction step
    static constexpr int kSliceRows = kRows / kSlices >= kStep ? kRows / kSlices : kStep;
    static constexpr int kDxTurns = kRows / 32 * IB / kBackWaves > 0 ? kRows / 32 * IB / kBackWaves : 1;  // a wave's 32 x 32 blocks of dx
    static constexpr int kSteps = kPo / 2;                                                                // reduction steps of dx
};

template <class T, int OB, int IB>
__global__ __launch_bounds__(kBackThreads, 2) void linear_back_kernel(LinearArgs a, float* db_work, int blocks) {
    using M = Back<T, OB, IB>;
    using Slope = typename M::Slope;
    constexpr int kE = M::kE, kQ = 16 / kE, kRows = M::kRows, kStages = M::kStages, kPieces2 = (kRows * M::kPo + kBackThreads - 1) / kBackThreads;
    using Piece = Vec<T, kE>;
    using SlopePiece = Vec<Slope, 16 / sizeof(Slope)>;
    __shared__ u32x4 lds[kStages][M::kTile];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, l32 = lane & 31;
    const int tiles = (int)((a.rows + kRows - 1) / kRows);
    int tile = blockIdx.x;
    const int po = (a.out + kE - 1) / kE, pi = (a.in + kE - 1) / kE, ps = a.out / (16 / (int)sizeof(Slope));
    const bool slopes = a.slope != nullptr;
    auto stage = [&](int to, int t) {
        const long long row0 = (long long)t * kRows;
        M::Dy::stage(lds[to], (const T*)a.dy, a.dy_ld, row0, a.rows, po);
        if (slopes) M::S::stage(lds[to] + M::kS, (const Slope*)a.slope, a.out, row0, a.rows, ps);
        M::X::stage(lds[to] + M::kX, (const T*)a.x, a.x_ld, row0, a.rows, pi);
    };
#pragma unroll
    for (int i = 0; i < kStages; i++) {
        M::Dy::clear(lds[i], po);
        M::S::clear(lds[i] + M::kS, ps);
        M::X::clear(lds[i] + M::kX, pi);
    }
    // dx: feature block wave % IB, the weights' column fragments
    const int fb = wave % IB * 32, rg = wave / IB;
    u32x4 w[M::kSteps];
    if (a.dx) {
        const int f = fb + feature_of<T>(l32);
#pragma unroll
        for (int s = 0; s < M::kSteps; s++) {
            Vec<T, kE> v;
#pragma unroll
            for (int e = 0; e < kE; e++) {
                const int n = (2 * s + half) * kE + e;
                v.e[e] = f < a.in && n < a.out ? ((const T*)a.w)[(long long)n * a.w_ld + f] : (T)0.f;
            }
            w[s] = __builtin_bit_cast(u32x4, v);
        }
    }
    // weight gradient: column block ib, row blocks ob + j kBackWaves / IB, rows slice ... of a tile
    const int ib = wave % IB * 32, slice = M::kSlices > 1 ? wave / M::kBlocks : 0, ob = M::kSlices > 1 ? (wave % M::kBlocks) / IB : wave / IB;
    f32x16 dw[M::kMine] = {};
    float sum[kPieces2][kE] = {};
#pragma unroll
    for (int i = 0; i < kStages - 1; i++)
        if (tile + i * blocks < tiles) stage(i, tile + i * blocks);
    int buf = 0;
    for (; tile < tiles; tile += blocks) {
        // this tile has landed when only the loads of the kStages - 2 behind it are left (without slopes there are fewer)
        constexpr int kFew = (kStages - 2) * (M::Dy::kN + M::X::kN), kAll = kFew + (kStages - 2) * M::S::kN;
        if (tile + (kStages - 2) * blocks >= tiles) landed<0>();
        else if (slopes) landed<kAll>();
        else landed<kFew>();
        const int next = buf == 0 ? kStages - 1 : buf - 1;
        if (tile + (kStages - 1) * blocks < tiles) stage(next, tile + (kStages - 1) * blocks);
        u32x4* t = lds[buf];
        const long long row0 = (long long)tile * kRows;
        const bool last = row0 + kRows > a.rows;
#pragma unroll
        for (int i = 0; i < kPieces2; i++) {  // dy -> dz in place
            const int s = threadIdx.x + i * kBackThreads;
            if (kRows * M::kPo % kBackThreads && s >= kRows * M::kPo) break;
            const int r = M::Dy::row_of(s), piece = M::Dy::piece_of(s);
            auto v = __builtin_bit_cast(Piece, t[s]);
            float f[kE];
#pragma unroll
            for (int e = 0; e < kE; e++) f[e] = to_f(v.e[e]);
            if (slopes) {
                constexpr int kPer = sizeof(Slope) * kE / 16, kSE = 16 / sizeof(Slope);
#pragma unroll
                for (int k = 0; k < kPer; k++) {
                    const auto q = __builtin_bit_cast(SlopePiece, t[M::kS + M::S::at(r, piece * kPer + k)]);
#pragma unroll
                    for (int e = 0; e < kSE; e++) f[k * kSE + e] *= to_slope<T>(q.e[e]);
                }
            }
            if (last && row0 + r >= a.rows)
#pragma unroll
                for (int e = 0; e < kE; e++) f[e] = 0.f;
#pragma unroll
            for (int e = 0; e < kE; e++) sum[i][e] += f[e];
            if (slopes || last) {
#pragma unroll
                for (int e = 0; e < kE; e++) v.e[e] = (T)f[e];
                t[s] = __builtin_bit_cast(u32x4, v);
            }
        }
        if (last)  // rows past the end repeat the last one: no x of theirs, be it an infinity, meets a zero dz
            for (int s = threadIdx.x; s < M::X::kCount; s += kBackThreads) if (row0 + M::X::row_of(s) >= a.rows) t[M::kX + s] = u32x4{0, 0, 0, 0};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (a.dx) {
#pragma unroll
            for (int i = 0; i < M::kDxTurns; i++) {
                const int r0 = (rg + i * (kBackWaves / IB)) * 32;
                if (r0 >= kRows) break;
                f32x16 acc = {};
#pragma unroll
                for (int s = 0; s < M::kSteps; s++) mfma(acc, w[s], t[M::Dy::at(r0 + l32, 2 * s + half)], T{});
                const long long row = row0 + r0 + l32;
                if (row < a.rows)
#pragma unroll
                    for (int q = 0; q < kQ; q++) {
                        const int feat = fb + piece_feature<T>(q, half);
                        if (feat >= a.in) continue;
                        float v[kE];
#pragma unroll
                        for (int j = 0; j < kE; j++) v[j] = acc[q * kE + j];
                        store_n<T, kE>((T*)a.dx + row * a.dx_ld + feat, a.in - feat, v);
                    }
            }
        }
#pragma unroll
        for (int s = 0; s < M::kSliceRows / M::kStep; s++) {
            const int m = slice * M::kSliceRows + s * M::kStep;
            if (M::kSlices * M::kSliceRows > kRows && m >= kRows) break;
            const u32x4 ff = M::X::template transposed<true>(t + M::kX, ib, m);
#pragma unroll
            for (int j = 0; j < M::kMine; j++) mfma(dw[j], ff, M::Dy::template transposed<false>(t, (ob + j * (kBackWaves / IB)) * 32, m), T{});
        }
        buf = buf == kStages - 1 ? 0 : buf + 1;
    }
    const long long part = (long long)blockIdx.x * M::kSlices + slice, weights = (long long)a.out * a.in;
#pragma unroll
    for (int j = 0; j < M::kMine; j++) {
        const int n = (ob + j * (kBackWaves / IB)) * 32 + l32;
        if (n >= a.out) continue;
#pragma unroll
        for (int q = 0; q < kQ; q++) {
            const int feat = ib + piece_feature<T>(q, half);
            if (feat >= a.in) continue;
            float v[kE];
#pragma unroll
            for (int e = 0; e < kE; e++) v[e] = dw[j][q * kE + e];
            store_n<float, kE>(a.work + part * weights + (long long)n * a.in + feat, a.in - feat, v);
        }
    }
    if (!a.db) return;
    __syncthreads();
    float* join = (float*)lds;
#pragma unroll
    for (int i = 0; i < kPieces2; i++) {
        const int s = threadIdx.x + i * kBackThreads;
        if (s < kRows * M::kPo)
#pragma unroll
            for (int e = 0; e < kE; e++) join[s * kE + e] = sum[i][e];
    }
    __syncthreads();
    for (int n = threadIdx.x; n < a.out; n += kBackThreads) {
        float s = 0.f;
        for (int r = 0; r < kRows; r++) s += join[M::Dy::at(r, n / kE) * kE + n % kE];
        db_work[(long long)blockIdx.x * a.out + n] = s;
    }
}

// ---- few rows: latency is everything. One 32 x 32 tile a workgroup, the reduction dealt out to its eight waves, fragments
// straight from memory (all of a wave's loads under way at once, no LDS and no barrier before the sums are joined). ----
template <class T, int ACT>
__device__ __forceinline__ void few_forward(const LinearArgs& a, const float* sums, long long row0, int feat0) {
    const int r = threadIdx.x >> 4, f = (threadIdx.x & 15) * 2;
    const long long row = row0 + r;
    if (row >= a.rows) return;
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int feat = feat0 + f + j;
        if (feat >= a.out) continue;
        float z = a.b ? to_f(((const T*)a.b)[feat]) : 0.f, s;
#pragma unroll
        for (int w = 0; w < 8; w++) z += sums[w * 1024 + r * 32 + f + j];
        float v = activate<ACT, sizeof(T) == 4>(z, s);
        if (a.slope) ((typename Elem<T>::Slope*)a.slope)[row * a.out + feat] = (typename Elem<T>::Slope)(s * Elem<T>::kSlopeScale);
        if (a.res) v += to_f(((const T*)a.res)[row * a.res_ld + feat]);
        ((T*)a.y)[row * a.y_ld + feat] = (T)v;
    }
}

template <class T>
__global__ __launch_bounds__(512) void linear_few_kernel(LinearArgs a, int tiles_n) {
    constexpr int kE = Elem<T>::kE, kAhead = 4;
    __shared__ float sums[8 * 1024];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, l32 = lane & 31;
    const long long row0 = (long long)(blockIdx.x / tiles_n) * 32;
    const int feat0 = (int)(blockIdx.x % tiles_n) * 32;
    const long long row = row0 + l32 < a.rows ? row0 + l32 : a.rows - 1;
    const int feat = feat0 + l32 < a.out ? feat0 + l32 : a.out - 1;
    const T *x = (const T*)a.x + row * a.x_ld, *w = (const T*)a.w + feat * a.w_ld;
    f32x16 acc = {};
    const bool whole = a.in % kE == 0;
    for (int k0 = wave * 2 * kE; k0 < a.in; k0 += 8 * 2 * kE * kAhead) {
        u32x4 fx[kAhead], fw[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int k = k0 + i * 8 * 2 * kE + half * kE;
            if (whole) {
                const bool in = k < a.in;
                const int at = in ? k : 0;
                fx[i] = __builtin_bit_cast(u32x4, load_n<T, kE>(x + at, kE));
                fw[i] = __builtin_bit_cast(u32x4, load_n<T, kE>(w + at, kE));
                if (!in) fx[i] = fw[i] = u32x4{0, 0, 0, 0};
            } else {
                fx[i] = __builtin_bit_cast(u32x4, load_end<T, kE>(x, k, a.in));
                fw[i] = __builtin_bit_cast(u32x4, load_end<T, kE>(w, k, a.in));
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; i++) mfma(acc, fw[i], fx[i], T{});
    }
#pragma unroll
    for (int q = 0; q < 16; q++) sums[wave * 1024 + l32 * 32 + 8 * (q >> 2) + 4 * half + (q & 3)] = acc[q];
    __syncthreads();
    switch (a.act) {
        case DRONE_ACTIVATION_RELU: few_forward<T, DRONE_ACTIVATION_RELU>(a, sums, row0, feat0); break;
        case DRONE_ACTIVATION_TANH: few_forward<T, DRONE_ACTIVATION_TANH>(a, sums, row0, feat0); break;
        case DRONE_ACTIVATION_SILU: few_forward<T, DRONE_ACTIVATION_SILU>(a, sums, row0, feat0); break;
        case DRONE_ACTIVATION_GELU: few_forward<T, DRONE_ACTIVATION_GELU>(a, sums, row0, feat0); break;
        default: few_forward<T, DRONE_ACTIVATION_NONE>(a, sums, row0, feat0);
    }
}

// Joins the partial sums of the weight and bias gradients in a fixed order, 32 values a workgroup, eight threads a value:
// every result is the same in every run.
template <class T>
__global__ __launch_bounds__(kJoinThreads) void linear_join_kernel(const float* work, const float* db_work, T* dw, T* db, long long weights, int out, int w_parts, int b_parts) {
    __shared__ float join[8][32];
    const int c = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const long long nw = dw ? weights : 0, all = nw + (db ? out : 0);
    for (long long first = (long long)blockIdx.x * 32; first < all; first += (long long)gridDim.x * 32) {  // (once, up to kJoinBlocks)
        const long long i = first + c;
        const bool is_w = i < nw;
        const long long at = is_w ? i : i - nw, step = is_w ? weights : out;
        const float* p = (is_w ? work : db_work) + at;
        const int parts = is_w ? w_parts : b_parts;
        float s = 0.f;
        if (i < all)
#pragma unroll 4
            for (int k = slice; k < parts; k += 8) s += p[k * step];
        join[slice][c] = s;
        __syncthreads();
        if (!slice && i < all) {
#pragma unroll
            for (int k = 1; k < 8; k++) s += join[k][c];
            if (is_w) dw[at] = (T)s; else db[at] = (T)s;
        }
        __syncthreads();
    }
}

template <class T, Product P, int BM, int BN, int WM, int WN>
int launch(const LinearArgs& a, long long nrows, long long nfeat, int parts, long long red_part, hipStream_t s, float* db_work = nullptr) {
    const int tiles_n = (int)((nfeat + BN - 1) / BN);
    const long long tiles = (nrows + BM - 1) / BM * tiles_n, units = tiles * parts;
    linear_kernel<T, P, BM, BN, WM, WN><<<(unsigned)((units + 7) / 8 * 8), WM * WN * 64, 0, s>>>(a, db_work, tiles_n, tiles, parts, red_part);
    return (int)hipGetLastError();
}

// Few rows: 32-row tiles, so that 1 024 envs make 32 workgroups and not 8.
bool few(long long rows, long long feats) { return (rows + 127) / 128 * ((feats + 127) / 128) < 128; }

template <class T, Product P>
int product(const LinearArgs& a, long long feats, hipStream_t s) {
    if (few(a.rows, feats)) {
        if (feats <= 32) return launch<T, P, 32, 32, 1, 1>(a, a.rows, feats, 1, 0, s);
        return launch<T, P, 32, 64, 1, 2>(a, a.rows, feats, 1, 0, s);
    }
    if (feats <= 32) return launch<T, P, 128, 32, 4, 1>(a, a.rows, feats, 1, 0, s);
    if (feats <= 64) return launch<T, P, 128, 64, 4, 1>(a, a.rows, feats, 1, 0, s);
    return launch<T, P, 128, 128, 2, 2>(a, a.rows, feats, 1, 0, s);
}

// The weight gradient's reduction over the rows is split into parts: enough workgroups to fill the 256 CUs (twice, unless
// the product is so small that joining the parts costs more than it), at least 128 rows each.
struct Split { int bm, bn, parts; };
Split split_of(long long rows, int in, int out) {
    Split r = {out <= 64 ? 64 : 128, in <= 64 ? 64 : 128, 1};
    const long long tiles = (long long)((out + r.bm - 1) / r.bm) * ((in + r.bn - 1) / r.bn), want = tiles <= 2 ? 256 : 512;
    long long parts = (want + tiles - 1) / tiles;
    const long long most = (rows + 127) / 128;
    if (parts > most) parts = most;
    r.parts = parts < 1 ? 1 : (int)parts;
    return r;
}

template <class T>
int weight_grad(const LinearArgs& a, float* db_work, const Split& sp, hipStream_t s) {
    constexpr int kK = kPieces * Elem<T>::kE;
    const long long part = ((a.rows + sp.parts - 1) / sp.parts + kK - 1) / kK * kK;
    if (sp.bm == 64 && sp.bn == 64) return launch<T, kWeight, 64, 64, 2, 2>(a, a.out, a.in, sp.parts, part, s, db_work);
    if (sp.bm == 64) return launch<T, kWeight, 64, 128, 2, 2>(a, a.out, a.in, sp.parts, part, s, db_work);
    if (sp.bn == 64) return launch<T, kWeight, 128, 64, 2, 2>(a, a.out, a.in, sp.parts, part, s, db_work);
    return launch<T, kWeight, 128, 128, 2, 2>(a, a.out, a.in, sp.parts, part, s, db_work);
}

template <class T, Product P, int BM, int BN, int WM, int WN, int PIECES, int STAGES>
int stream(const LinearArgs& a, long long nrows, long long nfeat, int parts, long long red_part, hipStream_t s) {
    const int tiles_n = (int)((nfeat + BN - 1) / BN);
    const long long tiles = (nrows + BM - 1) / BM * tiles_n, units = tiles * parts;
    linear_stream_kernel<T, P, BM, BN, WM, WN, PIECES, STAGES><<<(unsigned)((units + 7) / 8 * 8), WM * WN * 64, 0, s>>>(a, tiles_n, tiles, parts, red_part);
    return (int)hipGetLastError();
}

template <class T, Product P>
int stream_product(const LinearArgs& a, long long feats, hipStream_t s) {
    if (feats <= 64) return stream<T, P, 128, 64, 4, 1, 8, 2>(a, a.rows, feats, 1, 0, s);
    // 256 x 256 tiles where they fill the card: half the loads from L2 for each product (65536 x 1024 x 1024 bf16: 179 us, 213
    // with 128 x 128; deeper pipelines of 32-element steps: 190). f32 is bound by its matrix rate either way.
    if constexpr (sizeof(T) == 2) {
        if (feats >= 256 && (a.rows + 255) / 256 * ((feats + 255) / 256) >= 512 && (P == kForward ? a.in : a.out) >= 512) return stream<T, P, 256, 256, 4, 2, 8, 2>(a, a.rows, feats, 1, 0, s);
    }
    return stream<T, P, 128, 128, 2, 2, 8, 2>(a, a.rows, feats, 1, 0, s);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

constexpr int kDzParts = 512;

// Persistent workgroups: as many as stay on the card at once, in whole multiples of the feature groups for each XCD.
template <class T, int KS, int WF, bool RES>
int resident(const LinearArgs& a, hipStream_t s) {
    using M = Resident<T, KS, WF, RES>;
    const int groups = (a.out + WF * 32 - 1) / (WF * 32);
    const long long tiles = (a.rows + M::kRows - 1) / M::kRows;
    long long slots = 32 * M::kPerCu / groups;  // row tiles in work on each XCD
    if (slots < 1) slots = 1;
    // With fewer than eight tiles each there is nothing to keep under way (65536 x 64 x 64 f32, two tiles a workgroup: 21.6 us
    // against 16.8 of the tiled form; 262144 x 256 x 256 bf16, thirty-two: 101 against 133).
    if (tiles < 64 * slots) return -1;
    linear_resident_kernel<T, KS, WF, RES, M::kPerCu><<<(unsigned)(8 * slots * groups), kResidentWaves * 64, 0, s>>>(a, groups, (int)slots);
    return (int)hipGetLastError();
}

template <class T, int KS, bool RES>
int resident_wide(const LinearArgs& a, hipStream_t s) {
    if constexpr (KS <= 4) {
        if (a.out <= 32) return resident<T, KS, 1, RES>(a, s);
    }
    if constexpr (KS <= 8) {
        if (a.out <= 64) return resident<T, KS, 2, RES>(a, s);
    }
    if constexpr (KS <= 16) {
        if (a.out <= 128) return resident<T, KS, 4, RES>(a, s);
    }
    return resident<T, KS, 8, RES>(a, s);
}

template <class T>
int resident_any(const LinearArgs& a, hipStream_t s) {
    const int steps = (a.in / Elem<T>::kE + 1) / 2;
    auto go = [&](auto res) {
        constexpr bool kRes = decltype(res)::value;
        if (steps <= 4) return resident_wide<T, 4, kRes>(a, s);
        if (steps <= 8) return resident_wide<T, 8, kRes>(a, s);
        if (steps <= 16) return resident_wide<T, 16, kRes>(a, s);
        return resident_wide<T, 32, kRes>(a, s);
    };
    return a.res ? go(std::true_type{}) : go(std::false_type{});
}

template <class T>
int forward_any(const LinearArgs& a, hipStream_t s) {
    constexpr int kE = Elem<T>::kE;
    const bool pieces = a.in % kE == 0 && a.x_ld % kE == 0 && a.w_ld % kE == 0 && aligned16(a.x) && aligned16(a.w);
    const bool whole_res = !a.res || (a.out % kE == 0 && a.res_ld % kE == 0 && aligned16(a.res));
    if (pieces && whole_res && a.in * (int)sizeof(T) <= 1024) {
        const int rc = resident_any<T>(a, s);
        if (rc >= 0) return rc;
    }
    const int tiles_n = (a.out + 31) / 32;
    // One workgroup a CU at most: beyond, the tiled form's reuse wins (1 x 512 x 512 bf16: 4.8 against 7.0 us, 1024 x 20 x 64
    // f32: 4.0 against 5.8; 2048 x 512 x 512 bf16, 1024 workgroups: 13.5 against 9.2).
    if ((a.rows + 31) / 32 * tiles_n <= 256) {
        linear_few_kernel<T><<<(unsigned)((a.rows + 31) / 32 * tiles_n), 512, 0, s>>>(a, tiles_n);
        return (int)hipGetLastError();
    }
    if (pieces && a.out > 32 && !few(a.rows, a.out)) return stream_product<T, kForward>(a, a.out, s);
    return product<T, kForward>(a, a.out, s);
}

// The class of a width in blocks of 32: 2, 4, 8 (f32: up to 4), 0 where the one-pass gradient does not reach. Wider pairs than
// 16 blocks spill (131072 x 256 x 256 bf16, forward and gradient: 301 us in one pass, 226 in three).
template <class T>
int blocks_of(int n) { return n <= 64 ? 2 : n <= 128 ? 4 : n <= 256 && sizeof(T) == 2 ? 8 : 0; }

// f(OB, IB) as types, for the classes of out and in; false if there is none.
template <class T, class F>
bool visit_back(int out, int in, F f) {
    const int ob = blocks_of<T>(out), ib = blocks_of<T>(in);
    if (!ob || !ib || ob * ib > 16) return false;
    using Two = std::integral_constant<int, 2>;
    using Four = std::integral_constant<int, 4>;
    using Eight = std::integral_constant<int, 8>;
    if (ob == 2 && ib == 2) f(Two{}, Two{});
    else if (ob == 2 && ib == 4) f(Two{}, Four{});
    else if (ob == 4 && ib == 2) f(Four{}, Two{});
    else if (ob == 4 && ib == 4) f(Four{}, Four{});
    else if constexpr (sizeof(T) == 2) {
        if (ob == 2) f(Two{}, Eight{}); else f(Eight{}, Two{});
    }
    return true;
}

// Workgroups: one a CU, each with enough tiles that its partial sum of the weight gradient is not most of what it moves.
template <class M>
int back_blocks(long long rows, int in, int out) {
    const long long tiles = (rows + M::kRows - 1) / M::kRows, least = (long long)in * out >= 128 * 128 ? 4 : 1, b = (tiles + least - 1) / least;
    return b < 1 ? 1 : b > 256 ? 256 : (int)b;
}

// How a gradient is computed: one plan for the workspace's size and the launches. Pieces: rows of x and dy (and w) are whole,
// aligned 16-byte pieces, as they are or after dz and copies of x and w have been laid out so.
struct Plan {
    bool narrow, stream, pad;
    size_t dw, db, dz, x, w, bytes;  // offsets into the workspace: partial sums, then the laid-out operands
    int w_parts, db_parts;
    long long dz_rows;               // rows of one part of the dz pass
};

template <class T>
Plan plan_of(long long rows, int in, int out, bool pieces, bool slopes) {
    Plan p = {};
    const bool many = !few(rows, in > out ? in : out) || rows >= 4096;
    int narrow_parts = 0, narrow_blocks = 0;
    const bool is_narrow = visit_back<T>(out, in, [&](auto ob, auto ib) {
        using M = Back<T, decltype(ob)::value, decltype(ib)::value>;
        narrow_blocks = back_blocks<M>(rows, in, out);
        narrow_parts = narrow_blocks * M::kSlices;
    });
    p.narrow = is_narrow && rows && (pieces || many);
    p.stream = !p.narrow && rows && (in > 64 || out > 64) && in >= 16 && out >= 16 && !few(rows, in) && (pieces || many);
    p.pad = (p.narrow || p.stream) && !pieces;
    const Split sp = split_of(rows, in, out);
    p.w_parts = p.narrow ? narrow_parts : sp.parts;
    p.dz_rows = (rows + kDzParts - 1) / kDzParts;
    const bool own_db = p.stream || p.pad;  // the bias gradient comes from the dz pass
    p.db_parts = own_db ? (int)((rows + p.dz_rows - 1) / (p.dz_rows ? p.dz_rows : 1)) : p.narrow ? narrow_blocks : sp.parts;
    auto take = [&](size_t bytes) { const size_t at = p.bytes; p.bytes += (bytes + 255) / 256 * 256; return at; };
    p.dw = take((size_t)p.w_parts * in * out * 4);
    p.db = take((size_t)p.db_parts * out * 4);
    p.dz = take(own_db && (slopes || p.pad) ? (size_t)rows * whole_pieces<T>(out) * sizeof(T) : 0);
    p.x = take(p.pad ? (size_t)rows * whole_pieces<T>(in) * sizeof(T) : 0);
    p.w = take(p.pad ? (size_t)out * whole_pieces<T>(in) * sizeof(T) : 0);
    return p;
}

template <class T>
int pad(const void* from, long long ld, long long rows, int cols, T* to, hipStream_t s) {
    const int pieces = (int)(whole_pieces<T>(cols) / Elem<T>::kE);
    const long long blocks = (rows * pieces + 255) / 256;
    linear_pad_kernel<T><<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, s>>>((const T*)from, ld, rows, cols, to, pieces);
    return (int)hipGetLastError();
}

template <class T>
int backward_any(LinearArgs a, hipStream_t s) {
    constexpr int kE = Elem<T>::kE, kK = kPieces * kE;
    const bool pieces = a.in % kE == 0 && a.out % kE == 0 && a.x_ld % kE == 0 && a.dy_ld % kE == 0 && a.w_ld % kE == 0 && aligned16(a.x) && aligned16(a.dy) && aligned16(a.slope) && aligned16(a.w);
    const bool sums = a.dw || a.db;
    const Plan p = plan_of<T>(a.rows, a.in, a.out, pieces, a.slope != nullptr);
    // The input gradient alone needs no workspace. With one a wide layer streams all the same (65536 x 1024 x 1024 bf16: 524 us
    // in tiles, 262 streamed); a narrow one would form the weight gradient with it, an odd one lay out x.
    if (!sums && !(a.work && p.stream && !p.pad)) return a.rows ? product<T, kInput>(a, a.in, s) : 0;
    char* const work = (char*)a.work;
    float *const dw_work = (float*)(work + p.dw), *const db_work = (float*)(work + p.db);
    int rc = 0;
    if (p.stream || p.pad) {
        T* const dz = a.slope || p.pad ? (T*)(work + p.dz) : nullptr;
        if (dz || a.db) {
            const dim3 grid((unsigned)p.db_parts, (a.out + 32 * kE - 1) / (32 * kE));
            if (a.out % kE == 0) linear_dz_kernel<T, true><<<grid, 256, 0, s>>>(a, dz, whole_pieces<T>(a.out), a.db ? db_work : nullptr, p.dz_rows);
            else linear_dz_kernel<T, false><<<grid, 256, 0, s>>>(a, dz, whole_pieces<T>(a.out), a.db ? db_work : nullptr, p.dz_rows);
            if ((rc = (int)hipGetLastError())) return rc;
        }
        if (dz) { a.dy = dz; a.dy_ld = whole_pieces<T>(a.out); a.slope = nullptr; }
        if (p.pad) {
            if ((rc = pad<T>(a.x, a.x_ld, a.rows, a.in, (T*)(work + p.x), s))) return rc;
            a.x = work + p.x; a.x_ld = whole_pieces<T>(a.in);
        }
        if (p.stream && p.pad && a.dx) {
            if ((rc = pad<T>(a.w, a.w_ld, a.out, a.in, (T*)(work + p.w), s))) return rc;
            a.w = work + p.w; a.w_ld = whole_pieces<T>(a.in);
        }
    }
    a.work = dw_work;
    if (p.narrow) {
        LinearArgs b = a;
        if (p.pad) b.db = nullptr;
        visit_back<T>(a.out, a.in, [&](auto ob, auto ib) {
            constexpr int OB = decltype(ob)::value, IB = decltype(ib)::value;
            const int blocks = back_blocks<Back<T, OB, IB>>(a.rows, a.in, a.out);
            linear_back_kernel<T, OB, IB><<<blocks, kBackThreads, 0, s>>>(b, db_work, blocks);
            rc = (int)hipGetLastError();
        });
    } else if (p.stream) {
        if (a.dx && (rc = stream_product<T, kInput>(a, a.in, s))) return rc;
        if (a.dw) {
            const long long part = ((a.rows + p.w_parts - 1) / p.w_parts + kK - 1) / kK * kK;
            rc = stream<T, kWeight, 128, 128, 2, 2, 8, 2>(a, a.out, a.in, p.w_parts, part, s);
        }
    } else {
        if (a.dx && a.rows && (rc = product<T, kInput>(a, a.in, s))) return rc;
        rc = weight_grad<T>(a, db_work, split_of(a.rows, a.in, a.out), s);
    }
    if (rc || !sums) return rc;
    const long long weights = (long long)a.out * a.in, all = (a.dw ? weights : 0) + (a.db ? a.out : 0);
    linear_join_kernel<T><<<(unsigned)std::min((all + 31) / 32, kJoinBlocks), kJoinThreads, 0, s>>>(dw_work, db_work, (T*)a.dw, (T*)a.db, weights, a.out, p.w_parts, p.db_parts);
    return (int)hipGetLastError();
}

template <class T>
size_t work_bytes(long long rows, int in, int out) {  // (alignment and the activation are not known: room for any)
    size_t most = 0;
    for (int pieces = 0; pieces < 2; pieces++)
        for (int slopes = 0; slopes < 2; slopes++) {
            const size_t b = plan_of<T>(rows, in, out, pieces, slopes).bytes;
            most = b > most ? b : most;
        }
    return most;
}

}  // namespace

// One object file per element type (the Makefile compiles this file three times): DRONE_ELEM and its suffix.
#define DRONE_NAME2(a, b) a##b
#define DRONE_NAME(a, b) DRONE_NAME2(a, b)
int DRONE_NAME(linear_forward_, DRONE_ELEM_NAME)(const LinearArgs& a, hipStream_t s) { return a.rows ? forward_any<DRONE_ELEM>(a, s) : 0; }
int DRONE_NAME(linear_backward_, DRONE_ELEM_NAME)(const LinearArgs& a, hipStream_t s) { return backward_any<DRONE_ELEM>(a, s); }
size_t DRONE_NAME(linear_work_, DRONE_ELEM_NAME)(long long rows, int in, int out) { return work_bytes<DRONE_ELEM>(rows, in, out); }

}  // namespace drone
