// Shared helpers of the 8-bit kernels: what a code is, and how fp32 values become codes.
//
// A row is held as codes and one fp32 scale: amax = max(max|x|, 2^-100); int8: scale = amax / 127, code = rint(x * inv) with
// inv = fl32(127 / amax); e4m3: scale = amax / 448, code = e4m3(fl32(x * inv)) with inv = fl32(448 / amax).  The floor keeps
// inv finite: a row of zeros gets codes 0 and a scale of 2^-100 / top.  A row with an infinity or a NaN has no scale: it gets
// codes 0 and scale NaN, so that whoever reads the row sees NaN instead of a plausible number.
#pragma once

#include "esp_common.cuh"

namespace esp {

constexpr float kAmaxFloor = 7.888609052210118e-31f;      // 2^-100
constexpr float kInt8Top = 127.f, kE4m3Top = 448.f;

template <int CODE> struct CodeTop;
template <> struct CodeTop<ESP_CODE_INT8> { static constexpr float v = kInt8Top; };
template <> struct CodeTop<ESP_CODE_E4M3> { static constexpr float v = kE4m3Top; };

// max|x| travels as the bit pattern of |x|: unsigned order is the order of magnitudes, with infinity and then NaN on top,
// so a NaN is not lost on the way (fmaxf would drop it).
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Programmatic launch.  A kernel launched with the attribute may start before the one ahead of it in the stream has ended; it waits
// for that kernel's end and results here (every thread, before anything else that kernel may write or read).
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// From here on (once every CTA has passed or left) a kernel behind this one that was launched so may start.
__device__ __forceinline__ void grid_dependents_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// Launch of a kernel that begins with grid_dependency_wait.
template <typename... P, typename... A>
inline cudaError_t launch_early(void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t s, A... args) {
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid; cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cfg.attrs = &at; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// Limit, in SM cycles, of the waits for work of one's own that is still in flight after a wait has run out.  It is not the limit that
// esp_set_wait_limit_cycles sets: a short one ends waits for others early, but not those for copies that write this CTA's memory.
static __device__ const long long kDrainLimitCycles = 2000000000LL;

struct RowScale { float inv, scale; bool finite; };
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits, float top) {
    RowScale r;
    r.finite = amax_bits < 0x7f800000u;
    const float a = fmaxf(__uint_as_float(amax_bits), kAmaxFloor);       // fmaxf(NaN, floor) = floor: unused then
    r.inv = r.finite ? __fdiv_rn(top, a) : 0.f;
    r.scale = r.finite ? __fdiv_rn(a, top) : __uint_as_float(0x7fc00000u);
    return r;
}

// Four codes in one word, first value in the lowest byte.
// int8: one fused multiply-add against 1.5 * 2^23 rounds the EXACT product x * inv once, to an integer, ties to even (the
// sum lies where fp32 has a spacing of 1), and leaves the two's-complement code in the lowest byte of the result.
template <int CODE>
__device__ __forceinline__ uint32_t pack_codes4(const float* x, float inv, bool finite) {
    if (!finite) return 0u;
    if constexpr (CODE == ESP_CODE_INT8) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(__fmaf_rn(x[i], inv, 12582912.f));
        return __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
    } else {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(__fmul_rn(x[1], inv)), "f"(__fmul_rn(x[0], inv)));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(__fmul_rn(x[3], inv)), "f"(__fmul_rn(x[2], inv)));
        return (uint32_t)lo | ((uint32_t)hi << 16);
    }
}

// The four numbers that a word of codes holds (without the scale).
template <int CODE>
__device__ __forceinline__ void unpack_codes4(uint32_t w, float (&x)[4]) {
    if constexpr (CODE == ESP_CODE_INT8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t h;
            const uint16_t c = (uint16_t)(w >> (16 * i));
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
            const float2 f = Cvt<__half>::to_f2(h);
            x[2 * i] = f.x; x[2 * i + 1] = f.y;
        }
    }
}

}  // namespace esp
