// Row kernels around the 8-bit projections: residual add + RMSNorm, SiLU * mul, and the plain row quantiser, each with one
// fp32 scale per row (token) for its 8-bit form; and the way back.
//
//   add + norm   t = x + r (fp32); r <- round(t); y = t * rsqrt(mean(t^2) + eps) * w
//   SiLU * mul   y = g / (1 + exp(-g)) * u
//   codes        int8, scale = max|y| / 127 (quant_common.cuh)
// The norm is taken of the unrounded sum, so the output is rounded once; what is kept for the next layer is the rounded one.
//
// HBM bound: every element is read once, held in registers in fp32 (up to 8 * VPT per thread) across the row's reduction,
// and written once.  One CTA per row; the sum of squares and the maximum go through one shuffle + shared-memory reduction.
#include "quant_common.cuh"

namespace esp {

enum RowMode { ROW_ADD_NORM = 0, ROW_NORM = 1, ROW_SILU = 2, ROW_PLAIN = 3 };

struct RowArgs {
    const void* in; const void* weight; void* residual;      // in: [rows, cols] (ROW_SILU: [rows, 2*cols])
    int64_t in_stride;                                       // elements between rows of `in`
    void* out; int8_t* codes; float* scale;                  // one of out / codes
    int nvec;                                                // cols / 8
    float eps, inv_cols;
};

template <typename T, int MODE, int VPT, bool QUANT>
__global__ void __launch_bounds__(1024) row_kernel(RowArgs a) {
    const int64_t row = blockIdx.x;
    const int nt = blockDim.x;
    const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.in) + row * a.in_stride);
    uint4* res = MODE == ROW_ADD_NORM ? reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.residual) + row * (int64_t)a.nvec * 8) : nullptr;
    const uint4* wv = reinterpret_cast<const uint4*>(a.weight);
    constexpr bool kNorm = MODE == ROW_ADD_NORM || MODE == ROW_NORM;
    float t[VPT][8];
    uint4 v0[VPT], v1[VPT];
#pragma unroll
    for (int c = 0; c < VPT; ++c) {
        const int i = threadIdx.x + c * nt;
        if (i < a.nvec) {
            v0[c] = src[i];
            if (MODE == ROW_ADD_NORM) v1[c] = res[i];
            if (MODE == ROW_SILU) v1[c] = src[a.nvec + i];
        }
    }
    float ss = 0.f;
    uint32_t amax = 0;
#pragma unroll
    for (int c = 0; c < VPT; ++c) {
        const int i = threadIdx.x + c * nt;
        if (i < a.nvec) {
            const uint32_t u[4] = {v0[c].x, v0[c].y, v0[c].z, v0[c].w}, q[4] = {v1[c].x, v1[c].y, v1[c].z, v1[c].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float2 f = Cvt<T>::to_f2(u[k]);
                if (MODE == ROW_ADD_NORM) { const float2 g = Cvt<T>::to_f2(q[k]); f.x += g.x; f.y += g.y; }
                if (MODE == ROW_SILU) {
                    const float2 g = Cvt<T>::to_f2(q[k]);
                    f.x = __fdividef(f.x, 1.f + __expf(-f.x)) * g.x;
                    f.y = __fdividef(f.y, 1.f + __expf(-f.y)) * g.y;
                }
                if (kNorm) { ss = fmaf(f.x, f.x, ss); ss = fmaf(f.y, f.y, ss); }
                t[c][2 * k] = f.x; t[c][2 * k + 1] = f.y;
            }
            if (MODE == ROW_ADD_NORM)
                res[i] = make_uint4(Cvt<T>::pack(t[c][0], t[c][1]), Cvt<T>::pack(t[c][2], t[c][3]), Cvt<T>::pack(t[c][4], t[c][5]), Cvt<T>::pack(t[c][6], t[c][7]));
            if (kNorm) {
                const uint4 w = wv[i];
                const uint32_t g[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) { const float2 h = Cvt<T>::to_f2(g[k]); t[c][2 * k] *= h.x; t[c][2 * k + 1] *= h.y; }
            }
            if (QUANT) {
#pragma unroll
                for (int k = 0; k < 8; ++k) amax = max(amax, abs_bits(t[c][k]));
            }
        }
    }
    __shared__ float s_ss[32];
    __shared__ uint32_t s_mx[32];
    if (kNorm) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
    if (QUANT) amax = __reduce_max_sync(0xffffffffu, amax);
    const int warps = nt >> 5;
    if ((threadIdx.x & 31) == 0) { s_ss[threadIdx.x >> 5] = ss; s_mx[threadIdx.x >> 5] = amax; }
    __syncthreads();
    ss = 0.f; amax = 0;
    for (int i = 0; i < warps; ++i) { ss += s_ss[i]; amax = max(amax, s_mx[i]); }
    const float rstd = kNorm ? rsqrtf(fmaf(ss, a.inv_cols, a.eps)) : 1.f;
    if (QUANT) {
        // the maximum of |t * w * rstd| is that of |t * w| times rstd: rounding a product is monotonic
        const RowScale r = row_scale(abs_bits(__uint_as_float(amax) * rstd), kInt8Top);
        if (threadIdx.x == 0) a.scale[row] = r.scale;
        uint2* dst = reinterpret_cast<uint2*>(a.codes + row * (int64_t)a.nvec * 8);
#pragma unroll
        for (int c = 0; c < VPT; ++c) {
            const int i = threadIdx.x + c * nt;
            if (i < a.nvec) {
                float y[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = t[c][k] * rstd;
                dst[i] = make_uint2(pack_codes4<ESP_CODE_INT8>(y, r.inv, r.finite), pack_codes4<ESP_CODE_INT8>(y + 4, r.inv, r.finite));
            }
        }
    } else {
        uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + row * (int64_t)a.nvec * 8);
#pragma unroll
        for (int c = 0; c < VPT; ++c) {
            const int i = threadIdx.x + c * nt;
            if (i < a.nvec) {
                uint32_t o[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = Cvt<T>::pack(t[c][2 * k] * rstd, t[c][2 * k + 1] * rstd);
                dst[i] = make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
    }
}

// 16 codes per lane and step
template <typename OT>
__global__ void __launch_bounds__(256) dequantize_rows_kernel(OT* __restrict__ out, const int8_t* __restrict__ codes,
                                                              const float* __restrict__ scale, int64_t rows, int vecs) {
    const int64_t total = rows * vecs, stride = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += stride) {
        const uint2 w = reinterpret_cast<const uint2*>(codes)[i];
        const float s = scale[i / vecs];
        float f[4], g[4];
        unpack_codes4<ESP_CODE_INT8>(w.x, f); unpack_codes4<ESP_CODE_INT8>(w.y, g);
        if constexpr (sizeof(OT) == 4) {
            float4* o = reinterpret_cast<float4*>(out + i * 8);
            o[0] = make_float4(f[0] * s, f[1] * s, f[2] * s, f[3] * s);
            o[1] = make_float4(g[0] * s, g[1] * s, g[2] * s, g[3] * s);
        } else {
            *reinterpret_cast<uint4*>(out + i * 8) = make_uint4(Cvt<OT>::pack(f[0] * s, f[1] * s), Cvt<OT>::pack(f[2] * s, f[3] * s),
                                                               Cvt<OT>::pack(g[0] * s, g[1] * s), Cvt<OT>::pack(g[2] * s, g[3] * s));
        }
    }
}

constexpr int kMaxRowCols = 8 * 8 * 1024;          // VPT 8 x 1024 threads x 8 elements

template <typename T, int MODE, bool QUANT>
static int launch_row(RowArgs a, int64_t rows, int cols, cudaStream_t s) {
    a.nvec = cols / 8;
    a.inv_cols = 1.f / (float)cols;
    // 16-byte vectors per thread: 2 keeps a row of 4096 in 256 threads; wider rows hold more per thread up to 8
    const int vpt = a.nvec <= 2 * 512 ? 2 : (a.nvec <= 4 * 512 ? 4 : 8);
    int nt = ((a.nvec + vpt - 1) / vpt + 31) / 32 * 32;
    const unsigned grid = (unsigned)rows;
    if (vpt == 2) row_kernel<T, MODE, 2, QUANT><<<grid, nt, 0, s>>>(a);
    else if (vpt == 4) row_kernel<T, MODE, 4, QUANT><<<grid, nt, 0, s>>>(a);
    else row_kernel<T, MODE, 8, QUANT><<<grid, nt, 0, s>>>(a);
    ESP_LAUNCH_CHECK("row_kernel");
    return ESP_OK;
}

static int check_row(int64_t rows, int32_t cols, int32_t dtype) {
    if (rows < 0 || cols <= 0 || (dtype != ESP_DTYPE_F16 && dtype != ESP_DTYPE_BF16)) return ESP_ERR_BAD_ARG;
    if (cols % 8) return ESP_ERR_ALIGNMENT;
    if (cols > kMaxRowCols || rows > 2147483647LL) return ESP_ERR_TOO_LARGE;
    return ESP_OK;
}

}  // namespace esp

using namespace esp;

extern "C" int esp_add_rms_norm(void* out, void* residual, const void* in, const void* weight, int64_t tokens, int32_t hidden, float eps,
                                int32_t dtype, void* stream) {
    if (tokens == 0) return ESP_OK;
    if (!out || !residual || !in || !weight) return ESP_ERR_BAD_ARG;
    const int rc = check_row(tokens, hidden, dtype);
    if (rc) return rc;
    if (!aligned16(out) || !aligned16(residual) || !aligned16(in) || !aligned16(weight)) return ESP_ERR_ALIGNMENT;
    RowArgs a{in, weight, residual, hidden, out, nullptr, nullptr, 0, eps, 0.f};
    return dtype == ESP_DTYPE_F16 ? launch_row<__half, ROW_ADD_NORM, false>(a, tokens, hidden, (cudaStream_t)stream)
                                  : launch_row<__nv_bfloat16, ROW_ADD_NORM, false>(a, tokens, hidden, (cudaStream_t)stream);
}

extern "C" int esp_add_rms_norm_q8(int8_t* codes, float* scale, void* residual, const void* in, const void* weight, int64_t tokens,
                                   int32_t hidden, float eps, int32_t dtype, void* stream) {
    if (tokens == 0) return ESP_OK;
    if (!codes || !scale || !in || !weight) return ESP_ERR_BAD_ARG;
    const int rc = check_row(tokens, hidden, dtype);
    if (rc) return rc;
    if (!aligned16(codes) || !aligned16(residual) || !aligned16(in) || !aligned16(weight)) return ESP_ERR_ALIGNMENT;
    RowArgs a{in, weight, residual, hidden, nullptr, codes, scale, 0, eps, 0.f};
    cudaStream_t s = (cudaStream_t)stream;
    if (residual)
        return dtype == ESP_DTYPE_F16 ? launch_row<__half, ROW_ADD_NORM, true>(a, tokens, hidden, s)
                                      : launch_row<__nv_bfloat16, ROW_ADD_NORM, true>(a, tokens, hidden, s);
    return dtype == ESP_DTYPE_F16 ? launch_row<__half, ROW_NORM, true>(a, tokens, hidden, s)
                                  : launch_row<__nv_bfloat16, ROW_NORM, true>(a, tokens, hidden, s);
}

extern "C" int esp_silu_and_mul_q8(int8_t* codes, float* scale, const void* io, int64_t tokens, int32_t ffn_inter_dim, int32_t dtype,
                                   void* stream) {
    if (tokens == 0) return ESP_OK;
    if (!codes || !scale || !io) return ESP_ERR_BAD_ARG;
    const int rc = check_row(tokens, ffn_inter_dim, dtype);
    if (rc) return rc;
    if (!aligned16(codes) || !aligned16(io)) return ESP_ERR_ALIGNMENT;
    RowArgs a{io, nullptr, nullptr, 2 * (int64_t)ffn_inter_dim, nullptr, codes, scale, 0, 0.f, 0.f};
    return dtype == ESP_DTYPE_F16 ? launch_row<__half, ROW_SILU, true>(a, tokens, ffn_inter_dim, (cudaStream_t)stream)
                                  : launch_row<__nv_bfloat16, ROW_SILU, true>(a, tokens, ffn_inter_dim, (cudaStream_t)stream);
}

extern "C" int esp_quantize_rows(int8_t* codes, float* scale, const void* x, int64_t x_row_stride, int64_t rows, int32_t cols, int32_t dtype,
                                 void* stream) {
    if (rows == 0) return ESP_OK;
    if (!codes || !scale || !x) return ESP_ERR_BAD_ARG;
    const int rc = check_row(rows, cols, dtype);
    if (rc) return rc;
    if (!aligned16(codes) || !aligned16(x) || x_row_stride % 8) return ESP_ERR_ALIGNMENT;
    RowArgs a{x, nullptr, nullptr, x_row_stride, nullptr, codes, scale, 0, 0.f, 0.f};
    return dtype == ESP_DTYPE_F16 ? launch_row<__half, ROW_PLAIN, true>(a, rows, cols, (cudaStream_t)stream)
                                  : launch_row<__nv_bfloat16, ROW_PLAIN, true>(a, rows, cols, (cudaStream_t)stream);
}

extern "C" int esp_dequantize_rows(void* out, const int8_t* codes, const float* scale, int64_t rows, int32_t cols, int32_t dtype, void* stream) {
    if (rows == 0) return ESP_OK;
    if (!out || !codes || !scale || rows < 0 || cols <= 0) return ESP_ERR_BAD_ARG;
    if (cols % 8 || !aligned16(out) || ((uintptr_t)codes & 7u)) return ESP_ERR_ALIGNMENT;
    const int64_t want = (rows * (cols / 8) + 255) / 256, cap = (int64_t)kNumSMs * 32;
    const unsigned grid = (unsigned)(want < cap ? want : cap);
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == ESP_DTYPE_F16) dequantize_rows_kernel<__half><<<grid, 256, 0, s>>>((__half*)out, codes, scale, rows, cols / 8);
    else if (dtype == ESP_DTYPE_BF16) dequantize_rows_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>((__nv_bfloat16*)out, codes, scale, rows, cols / 8);
    else if (dtype == ESP_DTYPE_F32) dequantize_rows_kernel<float><<<grid, 256, 0, s>>>((float*)out, codes, scale, rows, cols / 8);
    else return ESP_ERR_BAD_ARG;
    ESP_LAUNCH_CHECK("dequantize_rows_kernel");
    return ESP_OK;
}
