// drone_policy.hpp — what the policy operators' translation units share: argument blocks of the launches, element types,
// 16-byte pieces. Internal to the library (include/drone_vec.h is the boundary).
#pragma once

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

namespace drone {

// y = act(x W^T + b) + residual and its gradient. Strides in elements; slope [rows][out] dense.
struct LinearArgs {
    long long rows;
    int in, out;
    const void* x;
    const void* w;
    const void* b;
    const void* res;
    const void* dy;
    void* y;
    void* slope;     // forward: written if not null; backward: read, null when the activation is the identity
    void* dx;
    void* dw;
    void* db;
    float* work;
    long long x_ld, w_ld, res_ld, y_ld, dy_ld, dx_ld;  // dw is dense
    int act;
};

struct NormArgs {
    long long rows;
    int width;
    const void* x;
    const void* block;
    const void* gate;
    const void* post;
    const void* pre;
    void* r;
    void* h;
    const void* dr;  // or null: zero
    const void* dh;  // or null: zero
    void* dx;
    void* dblock;
    void* dgate;
    void* dpost;
    void* dpre;
    float* work;
    long long x_ld, block_ld, gate_ld;  // r, h, dr, dh and the gradients are dense
    int gate_rows;   // 0: no gate, 1: one [width] gate for every row, 2: [rows][width]
    float scale, eps;
};

constexpr int kAdamwTensors = 40;  // tensors of one launch: their table travels in the kernel arguments (40 x 64 B of the 4 KiB), nothing to keep in HBM

struct AdamwTensor {
    void* p;            // 16-bit or 32-bit weight
    const void* g;
    float* m;
    float* v;
    float* master;      // 32-bit weight behind a 16-bit p, or null
    long long n;
    int first_chunk;    // of this launch
    int vec;            // all its pointers are 16-byte aligned
};

struct AdamwArgs {
    AdamwTensor t[kAdamwTensors];
    int count, chunks;
    int parts;          // partial sums of the norm, all launches together; 0: no clipping
    int part0;          // norm launches: where this launch's partials begin
    int advance;        // norm launch 0: step += 1
    float* partial;
    float* norm;        // [1] or null
    int* step;
    float lr, decay, b1, b2, rest1, rest2, eps, max_norm;  // decay = 1 - lr wd, rest = 1 - b: formed in 64 bits (1 - 0.999f is 1e-5 off)
    float log_b1, log_b2;
};

// Launchers: 0, or the hipError_t of the launch. All check nothing: drone_policy.cpp has.
#define DRONE_LINEAR_ENTRY(name)                                    \
    int linear_forward_##name(const LinearArgs& a, hipStream_t s);  \
    int linear_backward_##name(const LinearArgs& a, hipStream_t s); \
    size_t linear_work_##name(long long rows, int in, int out);
DRONE_LINEAR_ENTRY(f32)
DRONE_LINEAR_ENTRY(bf16)
DRONE_LINEAR_ENTRY(f16)
inline int linear_forward_launch(int dtype, const LinearArgs& a, hipStream_t s) { return dtype == 0 ? linear_forward_f32(a, s) : dtype == 1 ? linear_forward_bf16(a, s) : linear_forward_f16(a, s); }
inline int linear_backward_launch(int dtype, const LinearArgs& a, hipStream_t s) { return dtype == 0 ? linear_backward_f32(a, s) : dtype == 1 ? linear_backward_bf16(a, s) : linear_backward_f16(a, s); }
inline size_t linear_work_bytes(int dtype, long long rows, int in, int out) { return dtype == 0 ? linear_work_f32(rows, in, out) : dtype == 1 ? linear_work_bf16(rows, in, out) : linear_work_f16(rows, in, out); }
int norm_forward_launch(int dtype, const NormArgs& a, hipStream_t s);
int norm_backward_launch(int dtype, const NormArgs& a, hipStream_t s);
size_t norm_work_bytes(int dtype, long long rows, int width);
int adamw_norm_launch(int dtype, const AdamwArgs& a, int blocks, hipStream_t s);
int adamw_update_launch(int dtype, const AdamwArgs& a, hipStream_t s);
int adamw_small_launch(int dtype, const AdamwArgs& a, hipStream_t s);
constexpr int kAdamwSmall = 8;      // chunks up to which one workgroup does the whole step in one launch
constexpr int kAdamwChunk = 2048;   // elements one workgroup updates
constexpr int kAdamwParts = 512;    // partial sums of one norm launch at most

}  // namespace drone

#ifdef __HIPCC__
namespace drone {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// kE elements make a 16-byte piece; Slope: the type act'(z) is kept in between forward and backward, finer than T, so that a
// 16-bit layer's gradient carries only two roundings (dz into the matrix core, the result into memory). A bf16 layer's are fp16
// times kSlopeScale: slopes lie in [-0.13, 1.13], so the products stay below 37 100, and a saturated unit's slope keeps eleven
// bits down to 2^-29 (tanh: |z| = 10.7; without the scale 5.5, and nothing left from 10 on) and bf16's eight to 2^-32. fp16
// itself needs f32.
template <class T> struct Elem;
template <> struct Elem<float> { static constexpr int kE = 4; using Slope = float; static constexpr float kSlopeScale = 1.f; };
template <> struct Elem<__bf16> { static constexpr int kE = 8; using Slope = _Float16; static constexpr float kSlopeScale = 32768.f; };
template <> struct Elem<_Float16> { static constexpr int kE = 8; using Slope = float; static constexpr float kSlopeScale = 1.f; };

}  // namespace drone
#endif
