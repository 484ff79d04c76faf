// Product of 8-bit integer matrices with a scale for every token and every output channel:
//   out[m, n] = (sum_k a[m, k] * w[n, k]) * a_scale[m] * w_scale[n]
// a [M, K] int8 rows of tokens, w [N, K] int8 rows of output channels (both with K contiguous), 32-bit integer sums, one
// rounding to the output type.  K <= 131071 keeps every sum inside 32 bits (128 * 128 * K < 2^31).
//
// First form: 64 x 64 tiles on the integer dot-product units.
#include "quant_common.cuh"

namespace esp {

template <typename OT> __device__ __forceinline__ OT from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

struct MmArgs {
    void* out; int64_t ldo; const int8_t* a; int64_t lda; const float* a_scale; const int8_t* w; int64_t ldw; const float* w_scale;
    int64_t M, N; int K;
};

template <typename OT>
__global__ void __launch_bounds__(256) mm_w8a8_tile_kernel(MmArgs g) {
    __shared__ uint32_t sa[64][17], sw[64][17];                  // 64 rows x 64 bytes, padded against bank conflicts
    const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int lr = threadIdx.x >> 2, lc = threadIdx.x & 3;       // loader: row, 16-byte piece
    int acc[4][4] = {};
    for (int k0 = 0; k0 < g.K; k0 += 64) {
        uint4 va = make_uint4(0, 0, 0, 0), vw = va;
        const int k = k0 + lc * 16;
        if (k < g.K) {
            if (m0 + lr < g.M) va = *reinterpret_cast<const uint4*>(g.a + (m0 + lr) * g.lda + k);
            if (n0 + lr < g.N) vw = *reinterpret_cast<const uint4*>(g.w + (n0 + lr) * g.ldw + k);
        }
        __syncthreads();
        sa[lr][lc * 4] = va.x; sa[lr][lc * 4 + 1] = va.y; sa[lr][lc * 4 + 2] = va.z; sa[lr][lc * 4 + 3] = va.w;
        sw[lr][lc * 4] = vw.x; sw[lr][lc * 4 + 1] = vw.y; sw[lr][lc * 4 + 2] = vw.z; sw[lr][lc * 4 + 3] = vw.w;
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < 16; ++kk) {
            int x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) { x[i] = (int)sa[ty + 16 * i][kk]; y[i] = (int)sw[tx + 16 * i][kk]; }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(x[i], y[j], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + ty + 16 * i;
        if (m >= g.M) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t n = n0 + tx + 16 * j;
            if (n < g.N) reinterpret_cast<OT*>(g.out)[m * g.ldo + n] = from_f32<OT>((float)acc[i][j] * g.a_scale[m] * g.w_scale[n]);
        }
    }
}

}  // namespace esp

using namespace esp;

extern "C" int esp_mm_w8a8(void* out, int64_t out_row_stride, const int8_t* a, int64_t a_row_stride, const float* a_scale, const int8_t* w,
                           int64_t w_row_stride, const float* w_scale, int64_t m, int64_t n, int64_t k, int32_t out_dtype, void* stream) {
    if (m == 0 || n == 0) return ESP_OK;
    if (!out || !a || !a_scale || !w || !w_scale || m < 0 || n < 0 || k <= 0) return ESP_ERR_BAD_ARG;
    if (out_row_stride < n || a_row_stride < k || w_row_stride < k) return ESP_ERR_BAD_ARG;
    if (k % 16 || a_row_stride % 16 || w_row_stride % 16 || !aligned16(a) || !aligned16(w)) return ESP_ERR_ALIGNMENT;
    if (k > 131071 || m > 4194240 || n > 2147483647LL) return ESP_ERR_TOO_LARGE;
    const MmArgs g{out, out_row_stride, a, a_row_stride, a_scale, w, w_row_stride, w_scale, m, n, (int)k};
    const dim3 grid((unsigned)((n + 63) / 64), (unsigned)((m + 63) / 64));
    cudaStream_t s = (cudaStream_t)stream;
    if (out_dtype == ESP_DTYPE_F16) mm_w8a8_tile_kernel<__half><<<grid, 256, 0, s>>>(g);
    else if (out_dtype == ESP_DTYPE_BF16) mm_w8a8_tile_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(g);
    else if (out_dtype == ESP_DTYPE_F32) mm_w8a8_tile_kernel<float><<<grid, 256, 0, s>>>(g);
    else return ESP_ERR_BAD_ARG;
    ESP_LAUNCH_CHECK("mm_w8a8_tile_kernel");
    return ESP_OK;
}
