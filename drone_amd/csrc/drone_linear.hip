// drone_linear.hip — y = act(x W^T + b) + residual and its gradient, for the policy networks a device-resident learner runs
// between env steps. Three products, one tiled kernel:
//   forward  Y[m][n]  = sum_k X[m][k] W[n][k]      bias, activation, residual and act'(z) in the epilogue
//   input    DX[m][k] = sum_n DZ[m][n] W[n][k]     DZ = dy * act'(z), formed while the tile is staged
//   weight   DW[n][k] = sum_m DZ[m][n] X[m][k]     split over m, partial sums joined in a fixed order; db rides along
#include <hip/hip_runtime.h>

#include "drone_policy.hpp"

#include "../../include/drone_vec.h"

namespace drone {
namespace {

constexpr int kThreads = 256;
constexpr int kPieces = 8;  // 16-byte pieces of the reduction axis a tile row holds: 64 16-bit or 32 f32 elements

template <class T> __device__ __forceinline__ float to_f(T v) { return (float)v; }

// ---- activation: value and slope in 32 bits. PRECISE (f32 tensors): the math library's functions. 16-bit tensors: the
// hardware exp2 / rcp (1 ulp) are far below the result's own rounding, and erf is Abramowitz & Stegun 7.1.26
// (|error| <= 1.5e-7), whose exp(-z^2/2) is also what the slope needs. ----
template <bool PRECISE>
__device__ __forceinline__ float activate(float z, int act, float& slope) {
    switch (act) {
        case DRONE_ACTIVATION_RELU:
            slope = z > 0.f ? 1.f : 0.f;
            return z > 0.f ? z : (z != z ? z : 0.f);  // a NaN stays one
        case DRONE_ACTIVATION_TANH: {
            float a;
            if (PRECISE) {
                a = tanhf(z);
            } else {
                const float big = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __expf(2.f * z));
                const float small = z * (1.f - z * z * 0.33333334f);
                a = fabsf(z) < 0.03f ? small : big;
            }
            slope = 1.f - a * a;
            return a;
        }
        case DRONE_ACTIVATION_SILU: {
            const float s = PRECISE ? 1.f / (1.f + expf(-z)) : __builtin_amdgcn_rcpf(1.f + __expf(-z));
            slope = s * (1.f + z * (1.f - s));
            if (fabsf(z) > 80.f) {  // 0 * inf at the infinities: the limits instead
                slope = z > 0.f ? 1.f : 0.f;
                return z > 0.f ? z : 0.f;
            }
            return z * s;
        }
        case DRONE_ACTIVATION_GELU: {
            const float e = PRECISE ? expf(-0.5f * z * z) : __expf(-0.5f * z * z);
            float cdf;
            if (PRECISE) {
                cdf = 0.5f * (1.f + erff(z * 0.70710678f));
            } else {
                const float x = fabsf(z) * 0.70710678f;
                const float t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * x);
                const float p = t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
                const float half_tail = 0.5f * p * e;
                cdf = z >= 0.f ? 1.f - half_tail : half_tail;
            }
            const float pdf = e * 0.39894228f;
            if (fabsf(z) > 3e38f) {  // an infinity: 0 * inf below
                slope = z > 0.f ? 1.f : 0.f;
                return z > 0.f ? z : 0.f;
            }
            slope = cdf + z * pdf;
            return z * cdf;
        }
        default:
            slope = 1.f;
            return z;
    }
}

// ---- tiles in LDS: [row][8 pieces of 16 B], piece p of row r at p ^ swz(r): eight neighbouring rows read the same piece
// from eight different bank groups, and the transposing loader's lanes (four rows apart) write to eight as well ----
__device__ __forceinline__ int swz(int r) { return (r ^ (r >> 3)) & 7; }

template <class T>
__device__ __forceinline__ u32x4 pack(const float* f) {
    union { u32x4 u; T t[Elem<T>::kE]; } o;
#pragma unroll
    for (int e = 0; e < Elem<T>::kE; e++) o.t[e] = (T)f[e];
    return o.u;
}

// One operand as it lies in memory. CONTIG: [row][reduction]; otherwise [reduction][row]. With `slope` the element is
// v * slope (the dz of the gradient), formed in 32 bits and rounded once to T for the matrix core.
template <class T>
struct Operand {
    const T* p;
    long long ld;
    const typename Elem<T>::Slope* slope;  // dense companion with leading dimension slope_ld, or null
    long long slope_ld;
};

// Loads ROWS x 8 pieces of a [row][reduction] operand: thread t takes piece t % 8 of rows t / 8 + 32 i.
template <class T, int ROWS, bool VEC>
struct ContigTile {
    static constexpr int kE = Elem<T>::kE, kN = ROWS * kPieces / kThreads;
    u32x4 reg[kN];
    __device__ __forceinline__ void load(const Operand<T>& o, long long row0, long long rows, long long k0, long long kend) {
        const int t = threadIdx.x, c = t & 7;
        const long long k = k0 + c * kE;
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const long long r = row0 + (t >> 3) + i * (kThreads / 8);
            union { u32x4 u; T e[kE]; } v;
            v.u = u32x4{0, 0, 0, 0};
            if (r < rows && k < kend) {
                const T* p = o.p + r * o.ld + k;
                if (VEC) {
                    v.u = *(const u32x4*)p;
                } else {
#pragma unroll
                    for (int e = 0; e < kE; e++) if (k + e < kend) v.e[e] = p[e];
                }
                if (o.slope) {
                    const auto* q = o.slope + r * o.slope_ld + k;
                    float f[kE];
                    if (VEC) {
                        struct Slopes { typename Elem<T>::Slope e[kE]; };
                        const Slopes s = *(const Slopes*)__builtin_assume_aligned(q, 16);
#pragma unroll
                        for (int e = 0; e < kE; e++) f[e] = to_f(v.e[e]) * to_f(s.e[e]);
                    } else {
#pragma unroll
                        for (int e = 0; e < kE; e++) f[e] = k + e < kend ? to_f(v.e[e]) * to_f(q[e]) : 0.f;
                    }
                    v.u = pack<T>(f);
                }
            }
            reg[i] = v.u;
        }
    }
    __device__ __forceinline__ void store(u32x4* lds) const {
        const int t = threadIdx.x, c = t & 7;
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int r = (t >> 3) + i * (kThreads / 8);
            lds[r * kPieces + (c ^ swz(r))] = reg[i];
        }
    }
};

// Loads the same tile from a [reduction][row] operand: a thread takes kE reduction steps x 4 rows (kE loads of 4 elements)
// and turns them in registers, so the LDS tile and the fragment reads are those of the contiguous form.
template <class T, int ROWS, bool VEC>
struct TransTile {
    static constexpr int kE = Elem<T>::kE, kBlocks = ROWS / 4 * kPieces, kN = (kBlocks + kThreads - 1) / kThreads;
    struct Four { T e[4]; } reg[kN][kE];
    // add: the 32-bit dz of this thread's four rows is added up over the reduction (the bias gradient)
    __device__ __forceinline__ void load(const Operand<T>& o, long long row0, long long rows, long long k0, long long kend, bool add, float (&sum)[kN][4]) {
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int b = threadIdx.x + i * kThreads;
            const long long r = row0 + (b % (ROWS / 4)) * 4, k = k0 + b / (ROWS / 4) * kE;
#pragma unroll
            for (int e = 0; e < kE; e++) {
                Four v;
#pragma unroll
                for (int j = 0; j < 4; j++) v.e[j] = (T)0.f;
                if (b < kBlocks && k + e < kend && r < rows) {
                    const T* p = o.p + (k + e) * o.ld + r;
                    if (VEC) {
                        v = *(const Four*)__builtin_assume_aligned(p, sizeof(Four));
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; j++) if (r + j < rows) v.e[j] = p[j];
                    }
                    if (o.slope || add) {
                        struct S4 { typename Elem<T>::Slope e[4]; } s;
                        const auto* q = o.slope ? o.slope + (k + e) * o.slope_ld + r : nullptr;
                        if (VEC && q) s = *(const S4*)__builtin_assume_aligned(q, sizeof(S4));
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            float f = to_f(v.e[j]);
                            if (q) f *= VEC ? to_f(s.e[j]) : (r + j < rows ? to_f(q[j]) : 0.f);
                            if (add) sum[i][j] += f;
                            v.e[j] = (T)f;
                        }
                    }
                }
                reg[i][e] = v;
            }
        }
    }
    __device__ __forceinline__ void store(u32x4* lds) const {
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int b = threadIdx.x + i * kThreads;
            if (b >= kBlocks) break;
            const int r = (b % (ROWS / 4)) * 4, c = b / (ROWS / 4);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                union { u32x4 u; T t[kE]; } v;
#pragma unroll
                for (int e = 0; e < kE; e++) v.t[e] = reg[i][e].e[j];
                lds[(r + j) * kPieces + (c ^ swz(r + j))] = v.u;
            }
        }
    }
};

// D += A B^T over one pair of 16-byte pieces per lane (the lane's half of the wave picks the piece, so a step spans 32 B of
// the reduction axis). The order of the reduction inside a step is the same for both operands, which is all the product needs.
__device__ __forceinline__ void mfma(f32x16& d, const u32x4& a, const u32x4& b, float) {
#pragma unroll
    for (int e = 0; e < 4; e++) d = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(b[e]), d, 0, 0, 0);
}
__device__ __forceinline__ void mfma(f32x16& d, const u32x4& a, const u32x4& b, __bf16) {
    d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), d, 0, 0, 0);
}
__device__ __forceinline__ void mfma(f32x16& d, const u32x4& a, const u32x4& b, _Float16) {
    d = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), d, 0, 0, 0);
}

enum Product { kForward, kInput, kWeight };

template <class T, int ROWS, bool CONTIG, bool VEC> struct TileOf { using type = ContigTile<T, ROWS, VEC>; };
template <class T, int ROWS, bool VEC> struct TileOf<T, ROWS, false, VEC> { using type = TransTile<T, ROWS, VEC>; };

template <class S> struct FourOf { S e[4]; };

template <class S>
__device__ __forceinline__ void load4(const S* p, int left, bool vec, float* f) {
    if (vec) {
        const FourOf<S> v = *(const FourOf<S>*)__builtin_assume_aligned(p, sizeof(FourOf<S>));
#pragma unroll
        for (int j = 0; j < 4; j++) f[j] = to_f(v.e[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) f[j] = j < left ? to_f(p[j]) : 0.f;
    }
}

template <class S>
__device__ __forceinline__ void store4(S* p, int left, bool vec, const float* f) {
    if (vec) {
        FourOf<S> v;
#pragma unroll
        for (int j = 0; j < 4; j++) v.e[j] = (S)f[j];
        *(FourOf<S>*)__builtin_assume_aligned(p, sizeof(FourOf<S>)) = v;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) if (j < left) p[j] = (S)f[j];
    }
}

// BM x BN outputs a workgroup (rows x features), four waves WM x WN. The features are the matrix instruction's first
// operand, so a lane ends up with four neighbouring features of one row.
template <class T, Product P, bool VEC, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(kThreads) void linear_kernel(LinearArgs a, int tiles_n, long long tiles, long long red_part, int out_vec) {
    using Slope = typename Elem<T>::Slope;
    constexpr int kE = Elem<T>::kE, kK = kPieces * kE, TM = BM / WM / 32, TN = BN / WN / 32;
    static_assert(WM * WN * 64 == kThreads && TM >= 1 && TN >= 1, "four waves");
    __shared__ u32x4 lds[2][(BM + BN) * kPieces];

    // tile number: one contiguous eighth of the tiles per XCD (workgroups go round the eight XCDs), features fastest, so
    // the workgroups that share a row tile share its L2
    const long long per = (tiles + 7) / 8, tile = (long long)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per || tile >= tiles) return;
    const long long tm = tile / tiles_n;
    const int tn = (int)(tile - tm * tiles_n);

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
        red0 = (long long)blockIdx.y * red_part;
        red1 = red0 + red_part < a.rows ? red0 + red_part : a.rows;
    }
    const long long row0 = tm * BM, feat0 = (long long)tn * BN;

    typename TileOf<T, BM, P != kWeight, VEC>::type rt;
    typename TileOf<T, BN, P == kForward, VEC>::type ft;
    constexpr int kSums = (BM / 4 * kPieces + kThreads - 1) / kThreads, kNoSums = (BN / 4 * kPieces + kThreads - 1) / kThreads;
    float sum[kSums][4] = {}, no_sum[kNoSums][4];
    const bool want_db = P == kWeight && a.db && tn == 0;
    auto fetch = [&](long long k) {
        if constexpr (P == kWeight) rt.load(rowsop, row0, nrows, k, red1, want_db, sum); else rt.load(rowsop, row0, nrows, k, red1);
        if constexpr (P == kForward) ft.load(featop, feat0, nfeat, k, red1); else ft.load(featop, feat0, nfeat, k, red1, false, no_sum);
    };

    f32x16 acc[TN][TM] = {};
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, l32 = lane & 31;
    const int wrow = (wave / WN) * TM * 32, wfeat = (wave % WN) * TN * 32;

    fetch(red0);
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

#pragma unroll
    for (int m = 0; m < TM; m++) {
        const long long row = row0 + wrow + m * 32 + l32;
        if (row >= nrows) continue;
#pragma unroll
        for (int n = 0; n < TN; n++)
#pragma unroll
            for (int q = 0; q < 4; q++) {  // register 4 q + j of a lane: feature 8 q + 4 half + j
                const long long feat = feat0 + wfeat + n * 32 + q * 8 + half * 4;
                if (feat >= nfeat) continue;
                const int left = nfeat - feat < 4 ? (int)(nfeat - feat) : 4;
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; j++) v[j] = acc[n][m][4 * q + j];
                if (P == kForward) {
                    float b[4] = {0.f, 0.f, 0.f, 0.f}, s[4];
                    if (a.b) load4((const T*)a.b + feat, left, out_vec, b);
#pragma unroll
                    for (int j = 0; j < 4; j++) v[j] = activate<sizeof(T) == 4>(v[j] + b[j], a.act, s[j]);
                    if (a.slope) store4((Slope*)a.slope + row * a.out + feat, left, out_vec, s);
                    if (a.res) {
                        load4((const T*)a.res + row * a.res_ld + feat, left, out_vec, b);
#pragma unroll
                        for (int j = 0; j < 4; j++) v[j] += b[j];
                    }
                    store4((T*)a.y + row * a.y_ld + feat, left, out_vec, v);
                } else if (P == kInput) {
                    store4((T*)a.dx + row * a.dx_ld + feat, left, out_vec, v);
                } else {
                    store4(a.work + (long long)blockIdx.y * a.out * a.in + row * a.in + feat, left, out_vec, v);
                }
            }
    }
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
            if (threadIdx.x < BM && row0 + threadIdx.x < nrows) {
                float s = 0.f;
#pragma unroll
                for (int c = 0; c < kPieces; c++) s += join[c * BM + threadIdx.x];
                a.work[(long long)gridDim.y * a.out * a.in + (long long)blockIdx.y * a.out + row0 + threadIdx.x] = s;
            }
        }
    }
}

// Joins the partial sums of the weight and bias gradients, part by part in order: every result is the same in every run.
template <class T>
__global__ __launch_bounds__(kThreads) void linear_join_kernel(const float* work, T* dw, T* db, long long weights, int out, int parts) {
    const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
    const long long all = (dw ? weights : 0) + (db ? out : 0);
    if (i >= all) return;
    const bool is_w = dw && i < weights;
    const long long at = is_w ? i : i - (dw ? weights : 0), step = is_w ? weights : out;
    const float* p = is_w ? work + at : work + parts * weights + at;
    float s = 0.f;
    for (int k = 0; k < parts; k++) s += p[k * step];
    if (is_w) dw[at] = (T)s; else db[at] = (T)s;
}

bool aligned(const void* p, size_t bytes) { return ((uintptr_t)p % bytes) == 0; }

// Parts the weight gradient's reduction is split into: enough workgroups to fill the 256 CUs twice, at least 256 rows each.
int weight_parts(long long rows, int in, int out, int bm, int bn) {
    const long long tiles = (long long)((out + bm - 1) / bm) * ((in + bn - 1) / bn);
    long long parts = (512 + tiles - 1) / tiles, most = (rows + 255) / 256;
    if (parts > most) parts = most;
    return parts < 1 ? 1 : (int)parts;
}

int tile_of(long long n) { return n <= 32 ? 32 : n <= 64 ? 64 : 128; }

template <class T, Product P, bool VEC, int BM, int BN, int WM, int WN>
int launch(const LinearArgs& a, long long nrows, long long nfeat, int parts, long long red_part, int out_vec, hipStream_t s) {
    const int tiles_n = (int)((nfeat + BN - 1) / BN);
    const long long tiles = (nrows + BM - 1) / BM * tiles_n;
    const dim3 grid((unsigned)((tiles + 7) / 8 * 8), (unsigned)parts);
    linear_kernel<T, P, VEC, BM, BN, WM, WN><<<grid, kThreads, 0, s>>>(a, tiles_n, tiles, red_part, out_vec);
    return (int)hipGetLastError();
}

template <class T, bool VEC>
int forward(const LinearArgs& a, int out_vec, hipStream_t s) {
    switch (tile_of(a.out)) {
        case 32: return launch<T, kForward, VEC, 128, 32, 4, 1>(a, a.rows, a.out, 1, 0, out_vec, s);
        case 64: return launch<T, kForward, VEC, 128, 64, 4, 1>(a, a.rows, a.out, 1, 0, out_vec, s);
        default: return launch<T, kForward, VEC, 128, 128, 2, 2>(a, a.rows, a.out, 1, 0, out_vec, s);
    }
}

template <class T, bool VEC>
int input_grad(const LinearArgs& a, int out_vec, hipStream_t s) {
    switch (tile_of(a.in)) {
        case 32: return launch<T, kInput, VEC, 128, 32, 4, 1>(a, a.rows, a.in, 1, 0, out_vec, s);
        case 64: return launch<T, kInput, VEC, 128, 64, 4, 1>(a, a.rows, a.in, 1, 0, out_vec, s);
        default: return launch<T, kInput, VEC, 128, 128, 2, 2>(a, a.rows, a.in, 1, 0, out_vec, s);
    }
}

template <class T, bool VEC>
int weight_grad(const LinearArgs& a, int out_vec, int parts, hipStream_t s) {
    constexpr int kK = kPieces * Elem<T>::kE;
    const long long part = ((a.rows + parts - 1) / parts + kK - 1) / kK * kK;
    const int bm = tile_of(a.out), bn = tile_of(a.in);
    if (bm <= 64 && bn <= 64) return launch<T, kWeight, VEC, 64, 64, 2, 2>(a, a.out, a.in, parts, part, out_vec, s);
    if (bm <= 64) return launch<T, kWeight, VEC, 64, 128, 2, 2>(a, a.out, a.in, parts, part, out_vec, s);
    if (bn <= 64) return launch<T, kWeight, VEC, 128, 64, 2, 2>(a, a.out, a.in, parts, part, out_vec, s);
    return launch<T, kWeight, VEC, 128, 128, 2, 2>(a, a.out, a.in, parts, part, out_vec, s);
}

int parts_of(long long rows, int in, int out) { return weight_parts(rows, in, out, tile_of(out) <= 64 ? 64 : 128, tile_of(in) <= 64 ? 64 : 128); }

template <class T>
int forward_any(const LinearArgs& a, hipStream_t s) {
    constexpr int kE = Elem<T>::kE;
    const bool vec = a.in % kE == 0 && a.x_ld % kE == 0 && a.w_ld % kE == 0 && aligned(a.x, 16) && aligned(a.w, 16);
    const int ov = a.out % 4 == 0 && a.y_ld % 4 == 0 && aligned(a.y, 4 * sizeof(T)) && (!a.b || aligned(a.b, 4 * sizeof(T))) &&
                   (!a.res || (a.res_ld % 4 == 0 && aligned(a.res, 4 * sizeof(T)))) && (!a.slope || aligned(a.slope, 16));
    return vec ? forward<T, true>(a, ov, s) : forward<T, false>(a, ov, s);
}

template <class T>
int backward_any(const LinearArgs& a, hipStream_t s) {
    constexpr int kE = Elem<T>::kE;
    int rc = 0;
    const bool dy16 = a.out % kE == 0 && a.dy_ld % kE == 0 && aligned(a.dy, 16) && (!a.slope || aligned(a.slope, 16));
    const bool w4 = a.in % 4 == 0 && a.w_ld % 4 == 0 && aligned(a.w, 4 * sizeof(T));
    if (a.dx && a.rows) {
        const int ov = a.in % 4 == 0 && a.dx_ld % 4 == 0 && aligned(a.dx, 4 * sizeof(T));
        rc = dy16 && w4 ? input_grad<T, true>(a, ov, s) : input_grad<T, false>(a, ov, s);
        if (rc) return rc;
    }
    if (a.dw || a.db) {
        const bool dy4 = a.out % 4 == 0 && a.dy_ld % 4 == 0 && aligned(a.dy, 4 * sizeof(T)) && (!a.slope || aligned(a.slope, 4 * sizeof(typename Elem<T>::Slope)));
        const bool x4 = a.in % 4 == 0 && a.x_ld % 4 == 0 && aligned(a.x, 4 * sizeof(T));
        const int parts = parts_of(a.rows, a.in, a.out);
        rc = dy4 && x4 ? weight_grad<T, true>(a, a.in % 4 == 0, parts, s) : weight_grad<T, false>(a, a.in % 4 == 0, parts, s);
        if (rc) return rc;
        const long long weights = (long long)a.out * a.in, all = (a.dw ? weights : 0) + (a.db ? a.out : 0);
        linear_join_kernel<T><<<(unsigned)((all + kThreads - 1) / kThreads), kThreads, 0, s>>>(a.work, (T*)a.dw, (T*)a.db, weights, a.out, parts);
        rc = (int)hipGetLastError();
    }
    return rc;
}

}  // namespace

int linear_forward_launch(int dtype, const LinearArgs& a, hipStream_t s) {
    if (!a.rows) return 0;
    return dtype == DRONE_F32 ? forward_any<float>(a, s) : dtype == DRONE_BF16 ? forward_any<__bf16>(a, s) : forward_any<_Float16>(a, s);
}
int linear_backward_launch(int dtype, const LinearArgs& a, hipStream_t s) {
    return dtype == DRONE_F32 ? backward_any<float>(a, s) : dtype == DRONE_BF16 ? backward_any<__bf16>(a, s) : backward_any<_Float16>(a, s);
}
size_t linear_work_bytes(int, long long rows, int in, int out) {
    return (size_t)parts_of(rows, in, out) * ((size_t)in * out + out) * sizeof(float);
}

}  // namespace drone
