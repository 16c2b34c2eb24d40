// Arithmetic and tensor-core helpers of the attention kernels: paired FP32
// instructions, FP16 splits, swizzled operand descriptors, bounded waits.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "tcgen05.cuh"

namespace nb200 {
namespace tile {

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_huge_valf();

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// Two FP32 operations an instruction, each rounded to nearest.
__device__ __forceinline__ unsigned long long bits2(float2 a) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
    return r;
}
__device__ __forceinline__ float2 pair2(unsigned long long a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
    return pair2(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
    return pair2(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
    return pair2(r);
}

template <bool BF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (BF) {
        __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t *>(&v);
    } else {
        __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<uint32_t *>(&v);
    }
}

// x = hi + lo in FP16: 22 significand bits of each value within range
__device__ __forceinline__ void split2(float x0, float x1, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x0, x1);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x0 - f.x, x1 - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

// The powers of two that bring a row's largest absolute value to [2^12, 2^13)
// (an FP16 pair then keeps 22 bits of every value that matters beside it), and back.
__device__ __forceinline__ void row_scale(float most, float &up, float &down) {
    const int ex = most > 0.f ? min(max((int)((__float_as_uint(most) >> 23) & 255) - 127, -100), 100) : 0;
    up = __uint_as_float((uint32_t)(127 + 12 - ex) << 23);
    down = __uint_as_float((uint32_t)(127 - 12 + ex) << 23);
}

// Two FP16 values of two int8 codes, exactly: the code plus 128 put into the
// low bits of 1024.0 gives 1024 + 128 + code, from which 1152 is taken.  `u`
// holds four codes with their sign bits flipped; SEL picks the two bytes.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t i8x2_to_f16(uint32_t u) {
    const uint32_t w = __byte_perm(u, 0x64646464u, SEL);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&w), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t *>(&r);
}
// Sixteen codes to FP16, in order.
__device__ __forceinline__ void i8x16_to_f16(uint4 w, uint4 &a, uint4 &b) {
    const uint32_t u[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
    a = make_uint4(i8x2_to_f16<0x4140>(u[0]), i8x2_to_f16<0x4342>(u[0]), i8x2_to_f16<0x4140>(u[1]),
                   i8x2_to_f16<0x4342>(u[1]));
    b = make_uint4(i8x2_to_f16<0x4140>(u[2]), i8x2_to_f16<0x4342>(u[2]), i8x2_to_f16<0x4140>(u[3]),
                   i8x2_to_f16<0x4342>(u[3]));
}

constexpr int kTile = 128;   // rows of a tile

// 128-byte swizzled operands: rows of 128 bytes in atoms of 8 rows, a 16-byte
// piece c of row r at piece c ^ (r % 8).  K-major (Q, K): SBO = 1024 between
// 8-row groups.  MN-major (V, whose keys are the rows and whose dimensions run
// along them): SBO = 1024 between groups of 8 keys, LBO between chunks of 64
// dimensions.
__device__ __forceinline__ uint64_t desc_k(uint32_t a) {
    return (uint64_t)((a >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}
template <int ROWS>
__device__ __forceinline__ uint64_t desc_mn(uint32_t a) {
    return (uint64_t)((a >> 4) & 0x3FFF) | ((uint64_t)(ROWS * 128 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// Byte of 16-byte piece c of row r in a tile of ROWS rows of 16-bit values.
template <int ROWS>
__device__ __forceinline__ int piece_at(int r, int c) {
    return (c >> 3) * (ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}
// kind::f16, M = 128, f32 accumulator: types at bits 7 and 10 (0 f16, 1 bf16), B
// MN-major at bit 16, N / 8 at bit 17, M / 16 at bit 24.
__host__ __device__ constexpr uint32_t idesc(bool bf, bool b_mn, int n) {
    return (1u << 4) | ((uint32_t)bf << 7) | ((uint32_t)bf << 10) | ((uint32_t)b_mn << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}
// One lane of a converged warp, the same each time.  The products are issued
// under it: the compiler then knows that one thread runs and keeps their
// descriptors in uniform registers (under `lane == 0` an issue took about 100
// cycles, and the issues bounded the kernels).
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// D[tmem] (+)= A[tmem] x B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(desc), "r"(acc)
        : "memory");
}

__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, int x, int y, int z, int w,
                                            uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5}], [%6];" ::"r"(smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_addr(bar))
        : "memory");
}

// Bounded wait.  Where one runs out (never in working order) the CTA gives up: its
// copying threads stop, its other warps, whose lanes have to stay together for the
// warp-wide instructions, run on without waiting and write NaN, and the kernel
// raises its fault flag.
constexpr uint32_t kWaitLimit = 1u << 16;
__device__ __forceinline__ bool wait_phase(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
    const uint32_t a = smem_addr(bar);
    uint32_t done;
    // most phases have ended by the time they are asked for: a test first, since
    // try_wait may suspend the thread for longer
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(a), "r"(parity)
        : "memory");
    if (done) return true;
    if (*abort_flag) return false;
    for (uint32_t i = 0; i < kWaitLimit; ++i) {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(a), "r"(parity)
            : "memory");
        if (done) return true;
        if ((i & 255) == 255 && *abort_flag) return false;
    }
    *abort_flag = 1;
    return false;
}

// Registers move from the warpgroup of products, copies and conversions to the
// others; the sum over the CTA stays what it was at the launch.
template <int N>
__device__ __forceinline__ void more_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
// The 256 threads of one tile.
__device__ __forceinline__ void tile_sync(int w) { asm volatile("bar.sync %0, 256;" ::"r"(1 + w) : "memory"); }

}  // namespace tile
}  // namespace nb200
