// drone_norm.hip — the norms after and before a block of a policy, fused with the block's gate and residual scale:
//   n(a) = a / sqrt(mean(a^2) + eps)
//   r = x + scale * s * n(block) * post,  s = sigmoid(gate) (1 without a gate);   h = n(r) * pre
// and the gradient, with t = dr + dn(r)[dh * pre] and dn(a)[g] = (g - n(a) mean(g n(a))) / rms(a):
//   dx = t;  dgate = t * scale * n(block) * post * s (1 - s);  dblock = dn(block)[t * scale * s * post];
//   dpost = sum_rows t * scale * s * n(block);  dpre = sum_rows dh * n(r)
// One pass over memory each way, everything in between in 32-bit registers: 8 / 64 / 256 threads hold one row, by its width.
// Bound by memory: 65536 x 512 bf16 with a gate per row and channel, forward 61 us (336 MB, 5.5 TB/s with what the last cache
// still holds), gradient 107 + 5 us (537 MB, 5.0 TB/s); a copy moves 5.1.
// The backward pass reads x and forms r again rather than reading the rounded r: as many bytes, and no rounding in between.
#include <hip/hip_runtime.h>

#include "drone_policy.hpp"

#include "../../include/drone_vec.h"

namespace drone {
namespace {

constexpr int kThreads = 256;
constexpr int kJoinThreads = 1024;
constexpr int kGradBlocks = 1024;  // workgroups of the backward pass at most: each leaves one partial sum per column

// kE neighbouring elements as they lie in memory, zero past the row's end.
template <class T, bool VEC>
__device__ __forceinline__ u32x4 load_piece(const T* p, int c, int width) {
    constexpr int kE = Elem<T>::kE;
    union { u32x4 u; T e[kE]; } v;
    v.u = u32x4{0, 0, 0, 0};
    if (VEC) {
        if (c < width) v.u = *(const u32x4*)(p + c);
    } else {
#pragma unroll
        for (int e = 0; e < kE; e++) if (c + e < width) v.e[e] = p[c + e];
    }
    return v.u;
}

template <class T>
__device__ __forceinline__ void unpack(u32x4 u, float* f) {
    union { u32x4 u; T e[Elem<T>::kE]; } v;
    v.u = u;
#pragma unroll
    for (int e = 0; e < Elem<T>::kE; e++) f[e] = (float)v.e[e];
}

template <class T, bool VEC>
__device__ __forceinline__ void store_piece(T* p, int c, int width, const float* f) {
    constexpr int kE = Elem<T>::kE;
    if (VEC) {
        union { u32x4 u; T e[kE]; } v;
#pragma unroll
        for (int e = 0; e < kE; e++) v.e[e] = (T)f[e];
        if (c < width) *(u32x4*)(p + c) = v.u;
    } else {
#pragma unroll
        for (int e = 0; e < kE; e++) if (c + e < width) p[c + e] = (T)f[e];
    }
}

template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float plus_dpp(float v) {
    return v + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, ROWS, 0xf, false));
}

// Sum over the TPR threads of a row, the same in all of them: neighbours' registers (a shuffle through LDS for each of six
// steps, four sums a row, was a third of the backward pass), whole workgroups through `join` and two barriers.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* join) {
    v = plus_dpp<0xB1>(v);   // lane ^ 1
    v = plus_dpp<0x4E>(v);   // lane ^ 2
    v = plus_dpp<0x141>(v);  // the other four of eight
    if (TPR == 8) return v;
    v = plus_dpp<0x140>(v);       // the other eight of sixteen
    v = plus_dpp<0x142, 0xa>(v);  // lane 15 of rows 0 and 2 to rows 1 and 3
    v = plus_dpp<0x143, 0xc>(v);  // lane 31 to rows 2 and 3: lane 63 has all
    v = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63));
    if (TPR == 256) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) join[threadIdx.x >> 6] = v;
        __syncthreads();
        v = join[0] + join[1] + join[2] + join[3];
    }
    return v;
}

// (the hardware's exp2 and reciprocal, one unit in the last place each: 2e-7 of the result at most, and one instruction where a
// correctly rounded quotient is ten)
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }

// sigmoid(z) and 1 - sigmoid(z), each to a few units of its own last place: the gate's gradient is their product, and 1 - s of a
// wide open gate would cancel.
__device__ __forceinline__ void sigmoids(float z, float& s, float& rest) {
    const float e = __expf(-fabsf(z)), more = __builtin_amdgcn_rcpf(1.f + e), less = e * more;
    s = z < 0.f ? less : more;
    rest = z < 0.f ? more : less;
}

template <class T, int TPR, int NP, bool VEC>
__global__ __launch_bounds__(kThreads) void norm_forward_kernel(NormArgs a) {
    constexpr int kE = Elem<T>::kE, kRows = kThreads / TPR;
    __shared__ float join[4];
    const int t = threadIdx.x % TPR;
    const float inv_width = 1.f / (float)a.width;
    const long long step = (long long)gridDim.x * kRows;
    // every thread of a workgroup makes the same number of turns (the row sums of 256 threads have barriers)
    for (long long row0 = (long long)blockIdx.x * kRows; row0 < a.rows; row0 += step) {
        const long long row = row0 + threadIdx.x / TPR;
        const int width = row < a.rows ? a.width : 0;  // no columns: zeros in, nothing out
        float r[NP][kE], y[NP][kE], sum = 0.f;
        u32x4 px[NP], pb[NP], pg[NP], pp[NP], pq[NP];  // everything the row needs is asked for first
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int c = (i * TPR + t) * kE;
            px[i] = load_piece<T, VEC>((const T*)a.x + row * a.x_ld, c, width);
            if (a.block) pb[i] = load_piece<T, VEC>((const T*)a.block + row * a.block_ld, c, width);
            if (a.gate_rows) pg[i] = load_piece<T, VEC>((const T*)a.gate + (a.gate_rows == 2 ? row * a.gate_ld : 0), c, width);
            if (a.post) pq[i] = load_piece<T, VEC>((const T*)a.post, c, width);
            if (a.pre) pp[i] = load_piece<T, VEC>((const T*)a.pre, c, width);
        }
#pragma unroll
        for (int i = 0; i < NP; i++) {
            unpack<T>(px[i], r[i]);
            if (!a.block) continue;
            unpack<T>(pb[i], y[i]);
#pragma unroll
            for (int e = 0; e < kE; e++) sum += y[i][e] * y[i][e];
        }
        if (a.block) {
            const float inv = 1.f / sqrtf(row_sum<TPR>(sum, join) * inv_width + a.eps);
#pragma unroll
            for (int i = 0; i < NP; i++) {
                float f[kE];
                if (a.post) {
                    unpack<T>(pq[i], f);
#pragma unroll
                    for (int e = 0; e < kE; e++) y[i][e] *= f[e];
                }
                if (a.gate_rows) {
                    unpack<T>(pg[i], f);
#pragma unroll
                    for (int e = 0; e < kE; e++) y[i][e] *= sigmoid(f[e]);
                }
#pragma unroll
                for (int e = 0; e < kE; e++) r[i][e] += a.scale * (inv * y[i][e]);
            }
        }
        if (a.r)
#pragma unroll
            for (int i = 0; i < NP; i++) store_piece<T, VEC>((T*)a.r + row * a.width, (i * TPR + t) * kE, width, r[i]);
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < NP; i++)
#pragma unroll
            for (int e = 0; e < kE; e++) sum += r[i][e] * r[i][e];
        const float inv = 1.f / sqrtf(row_sum<TPR>(sum, join) * inv_width + a.eps);
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int c = (i * TPR + t) * kE;
            float f[kE];
            if (a.pre) {
                unpack<T>(pp[i], f);
#pragma unroll
                for (int e = 0; e < kE; e++) f[e] *= inv * r[i][e];
            } else {
#pragma unroll
                for (int e = 0; e < kE; e++) f[e] = inv * r[i][e];
            }
            store_piece<T, VEC>((T*)a.h + row * a.width, c, width, f);
        }
    }
}

// Column sums of one workgroup (its row groups joined in order) into its row of the partial sums.
template <int TPR, int NP, int kE>
__device__ __forceinline__ void column_sum(const float (&acc)[NP][kE], float* out, int width, float* buf) {
    constexpr int kRows = kThreads / TPR, kCols = TPR * NP * kE;
    const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NP; i++)
#pragma unroll
        for (int e = 0; e < kE; e++) buf[g * kCols + (i * TPR + t) * kE + e] = acc[i][e];
    __syncthreads();
    for (int c = threadIdx.x; c < kCols && c < width; c += kThreads) {
        float s = 0.f;
        for (int k = 0; k < kRows; k++) s += buf[k * kCols + c];
        out[c] = s;
    }
}

template <class T, int TPR, int NP, bool VEC>
__global__ __launch_bounds__(kThreads) void norm_backward_kernel(NormArgs a) {
    constexpr int kE = Elem<T>::kE, kRows = kThreads / TPR;
    __shared__ float join[4];
    __shared__ float buf[kThreads * NP * kE];
    const int t = threadIdx.x % TPR;
    const float inv_width = 1.f / (float)a.width;
    const long long step = (long long)gridDim.x * kRows;
    float post_sum[NP][kE] = {}, pre_sum[NP][kE] = {}, gate_sum[NP][kE] = {};
    // what every row shares stays in registers; a row's own values are asked for while the row before it is worked on
    u32x4 w_post[NP], w_pre[NP], w_gate[NP], x_[NP], block_[NP], gate_[NP], dr_[NP], dh_[NP];
#pragma unroll
    for (int i = 0; i < NP; i++) {
        const int c = (i * TPR + t) * kE;
        if (a.post) w_post[i] = load_piece<T, VEC>((const T*)a.post, c, a.width);
        if (a.pre) w_pre[i] = load_piece<T, VEC>((const T*)a.pre, c, a.width);
        if (a.gate_rows == 1) w_gate[i] = load_piece<T, VEC>((const T*)a.gate, c, a.width);
        dr_[i] = dh_[i] = u32x4{0, 0, 0, 0};
    }
    auto ask = [&](long long row) {
        const int width = row < a.rows ? a.width : 0;
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int c = (i * TPR + t) * kE;
            x_[i] = load_piece<T, VEC>((const T*)a.x + row * a.x_ld, c, width);
            if (a.block) block_[i] = load_piece<T, VEC>((const T*)a.block + row * a.block_ld, c, width);
            if (a.gate_rows == 2) gate_[i] = load_piece<T, VEC>((const T*)a.gate + row * a.gate_ld, c, width);
            if (a.dh) dh_[i] = load_piece<T, VEC>((const T*)a.dh + row * a.width, c, width);
            if (a.dr) dr_[i] = load_piece<T, VEC>((const T*)a.dr + row * a.width, c, width);
        }
    };
    const long long first = (long long)blockIdx.x * kRows;
    if (first < a.rows) ask(first + threadIdx.x / TPR);
    for (long long row0 = first; row0 < a.rows; row0 += step) {
        const long long row = row0 + threadIdx.x / TPR;
        const int width = row < a.rows ? a.width : 0;
        // 1 / rms of the row; 0 behind the last one, whose zeros may add nothing to the column sums (without eps: 0 * inf)
        auto inverse = [&](float squares) { return width ? 1.f / sqrtf(squares * inv_width + a.eps) : 0.f; };
        float r[NP][kE], nb[NP][kE], s[NP][kE], rest[NP][kE], dh[NP][kE], d_[NP][kE], f[kE], sum = 0.f;
#pragma unroll
        for (int i = 0; i < NP; i++) {
            unpack<T>(x_[i], r[i]);
            unpack<T>(dh_[i], dh[i]);
            unpack<T>(dr_[i], d_[i]);
            if (!a.block) continue;
            unpack<T>(block_[i], nb[i]);
            if (a.gate_rows) unpack<T>(a.gate_rows == 2 ? gate_[i] : w_gate[i], s[i]);
#pragma unroll
            for (int e = 0; e < kE; e++) {
                sum += nb[i][e] * nb[i][e];
                if (a.gate_rows) sigmoids(s[i][e], s[i][e], rest[i][e]); else { s[i][e] = 1.f; rest[i][e] = 0.f; }
            }
        }
        if (row0 + step < a.rows) ask(row + step);
        float inv_b = 0.f;
        if (a.block) {
            inv_b = inverse(row_sum<TPR>(sum, join));
#pragma unroll
            for (int i = 0; i < NP; i++) {
                if (a.post) unpack<T>(w_post[i], f);
#pragma unroll
                for (int e = 0; e < kE; e++) {
                    nb[i][e] *= inv_b;
                    r[i][e] += a.scale * (s[i][e] * (nb[i][e] * (a.post ? f[e] : 1.f)));
                }
            }
        }
        float rr = 0.f, gr = 0.f;
#pragma unroll
        for (int i = 0; i < NP; i++) {
            if (a.pre) unpack<T>(w_pre[i], f);
#pragma unroll
            for (int e = 0; e < kE; e++) {
                rr += r[i][e] * r[i][e];
                gr += r[i][e] * dh[i][e] * (a.pre ? f[e] : 1.f);
            }
        }
        const float inv_r = inverse(row_sum<TPR>(rr, join));
        const float mean_gr = row_sum<TPR>(gr, join) * inv_width * inv_r;  // mean(dh * pre * n(r))
        float ub = 0.f;
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int c = (i * TPR + t) * kE;
            float d[kE], fp[kE], fq[kE];
            if (a.pre) unpack<T>(w_pre[i], fp);
            if (a.post) unpack<T>(w_post[i], fq);
#pragma unroll
            for (int e = 0; e < kE; e++) {
                const float n = r[i][e] * inv_r;
                pre_sum[i][e] += dh[i][e] * n;
                d[e] = d_[i][e] + inv_r * (dh[i][e] * (a.pre ? fp[e] : 1.f) - n * mean_gr);
                r[i][e] = d[e];  // t
            }
            if (a.dx) store_piece<T, VEC>((T*)a.dx + row * a.width, c, width, d);
            if (!a.block) continue;
#pragma unroll
            for (int e = 0; e < kE; e++) {
                const float td = r[i][e] * a.scale, u = td * s[i][e], w = a.post ? fq[e] : 1.f;
                post_sum[i][e] += u * nb[i][e];
                const float dg = u * (nb[i][e] * w) * rest[i][e];
                gate_sum[i][e] += dg;
                d[e] = dg;
                r[i][e] = u * w;
                ub += r[i][e] * nb[i][e];
            }
            if (a.dgate && a.gate_rows == 2) store_piece<T, VEC>((T*)a.dgate + row * a.width, c, width, d);
        }
        if (a.dblock) {
            const float mean_ub = row_sum<TPR>(ub, join) * inv_width;
#pragma unroll
            for (int i = 0; i < NP; i++) {
#pragma unroll
                for (int e = 0; e < kE; e++) f[e] = inv_b * (r[i][e] - nb[i][e] * mean_ub);
                store_piece<T, VEC>((T*)a.dblock + row * a.width, (i * TPR + t) * kE, width, f);
            }
        }
    }
    float* out = a.work + (long long)blockIdx.x * 3 * a.width;
    if (a.dpost) column_sum<TPR, NP, kE>(post_sum, out, a.width, buf);
    if (a.dpre) column_sum<TPR, NP, kE>(pre_sum, out + a.width, a.width, buf);
    if (a.dgate && a.gate_rows == 1) column_sum<TPR, NP, kE>(gate_sum, out + 2 * a.width, a.width, buf);
}

// Joins the workgroups' column sums in a fixed order: 32 columns a workgroup, 32 threads a column.
template <class T>
__global__ __launch_bounds__(kJoinThreads) void norm_join_kernel(const float* work, T* dpost, T* dpre, T* dgate, int width, int parts) {
    constexpr int kSlices = kJoinThreads / 32;
    __shared__ float join[kSlices][32];
    const int which = blockIdx.y, c = blockIdx.x * 32 + (threadIdx.x & 31), k0 = threadIdx.x >> 5;
    T* out = which == 0 ? dpost : which == 1 ? dpre : dgate;
    if (!out) return;
    float s = 0.f;
    if (c < width)
#pragma unroll 8
        for (int k = k0; k < parts; k += kSlices) s += work[((long long)k * 3 + which) * width + c];
    join[k0][threadIdx.x & 31] = s;
    __syncthreads();
    if (k0 || c >= width) return;
#pragma unroll
    for (int k = 1; k < kSlices; k++) s += join[k][threadIdx.x];
    out[c] = (T)s;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int grad_blocks(long long rows, int rows_per_block) {
    const long long b = (rows + rows_per_block - 1) / rows_per_block;
    return b < 1 ? 1 : b > kGradBlocks ? kGradBlocks : (int)b;
}

template <class T, int TPR, int NP, bool VEC>
int run(const NormArgs& a, bool backward, hipStream_t s) {
    constexpr int kRows = kThreads / TPR;
    if (!backward) {
        long long blocks = (a.rows + kRows - 1) / kRows;
        if (blocks > 8192) blocks = 8192;
        norm_forward_kernel<T, TPR, NP, VEC><<<(unsigned)blocks, kThreads, 0, s>>>(a);
        return (int)hipGetLastError();
    }
    const int blocks = grad_blocks(a.rows, kRows);
    norm_backward_kernel<T, TPR, NP, VEC><<<blocks, kThreads, 0, s>>>(a);
    int rc = (int)hipGetLastError();
    T* dgate = a.gate_rows == 1 ? (T*)a.dgate : nullptr;
    if (rc || !(a.dpost || a.dpre || dgate)) return rc;
    norm_join_kernel<T><<<dim3((a.width + 31) / 32, 3), kJoinThreads, 0, s>>>(a.work, (T*)a.dpost, (T*)a.dpre, dgate, a.width, blocks);
    return (int)hipGetLastError();
}

template <class T, bool VEC>
int by_width(const NormArgs& a, bool backward, hipStream_t s) {
    constexpr int kE = Elem<T>::kE;
    if (a.width <= 8 * kE) return run<T, 8, 1, VEC>(a, backward, s);
    if (a.width <= 64 * kE) return run<T, 64, 1, VEC>(a, backward, s);
    if (a.width <= 128 * kE) return run<T, 64, 2, VEC>(a, backward, s);
    if (a.width <= 256 * kE) return run<T, 256, 1, VEC>(a, backward, s);
    if (a.width <= 512 * kE) return run<T, 256, 2, VEC>(a, backward, s);
    return run<T, 256, 4, VEC>(a, backward, s);  // up to 1024 pieces: 4096 f32 (kNormMaxWidth)
}

template <class T>
int any(const NormArgs& a, bool backward, hipStream_t s) {
    constexpr int kE = Elem<T>::kE;
    const bool vec = a.width % kE == 0 && a.x_ld % kE == 0 && aligned16(a.x) && (!a.block || (a.block_ld % kE == 0 && aligned16(a.block))) &&
                     (a.gate_rows != 2 || a.gate_ld % kE == 0) && aligned16(a.gate) && aligned16(a.post) && aligned16(a.pre) &&
                     aligned16(a.r) && aligned16(a.h) && aligned16(a.dr) && aligned16(a.dh) && aligned16(a.dx) && aligned16(a.dblock) &&
                     aligned16(a.dgate) && aligned16(a.dpost) && aligned16(a.dpre);
    return vec ? by_width<T, true>(a, backward, s) : by_width<T, false>(a, backward, s);
}

int dispatch(int dtype, const NormArgs& a, bool backward, hipStream_t s) {
    return dtype == DRONE_F32 ? any<float>(a, backward, s) : dtype == DRONE_BF16 ? any<__bf16>(a, backward, s) : any<_Float16>(a, backward, s);
}

}  // namespace

int norm_forward_launch(int dtype, const NormArgs& a, hipStream_t s) { return a.rows ? dispatch(dtype, a, false, s) : 0; }
int norm_backward_launch(int dtype, const NormArgs& a, hipStream_t s) { return dispatch(dtype, a, true, s); }

size_t norm_work_bytes(int dtype, long long rows, int width) {
    const int e = dtype == DRONE_F32 ? 4 : 8;
    return (size_t)grad_blocks(rows, width <= 8 * e ? 32 : width <= 128 * e ? 4 : 1) * 3 * width * sizeof(float);
}

}  // namespace drone
