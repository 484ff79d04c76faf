// Row kernels around the 8-bit projections: residual add + RMSNorm, SiLU * mul, and the plain row quantiser, each with one
// fp32 scale per row (token) for its 8-bit form; and the way back.
//
//   add + norm   t = x + r (fp32); r <- round(t); y = t * rsqrt(mean(t^2) + eps) * w
//   SiLU * mul   y = g / (1 + exp(-g)) * u
//   codes        int8, scale = max|y| / 127 (quant_common.cuh)
// The norm is taken of the unrounded sum, so the output is rounded once; what is kept for the next layer is the rounded one.
//
// HBM bound: every element is read once, held in fp32 (8 * VPT per thread; in registers up to 16384 wide) across the row's reduction,
// and written once.  Rows of up to 512 elements: a warp per row, eight rows to a CTA, the next row asked for before the one in hand
// is reduced (60000 rows of 256 into codes: a CTA of one warp per row took 33 us, this form 10).  Wider rows: a CTA per row; asking for
// the next row there cost more in registers than it gained.  Measured (B200): add + norm into codes 16384 x 4096 70.5 us for 470 MB,
// SiLU * mul into codes 8192 x 11008 71.7 us for 451 MB, plain rows into codes 16384 x 4096 38.8 us and back 34.0 us for 201 MB.
// Rows wider than 16384 (VPT 8) are compiled for 1024 threads and do not fit the registers that this leaves: 60 to 220 bytes per thread
// go through local memory, with the residual add 820.  4096 x 28672: SiLU * mul 127 us (0.71 of the copy rate), plain rows 76 (0.71), add +
// norm 415 (0.30).
#include "quant_common.cuh"
#include "sm100_ptx.cuh"

namespace esp {

enum RowMode { ROW_ADD_NORM = 0, ROW_NORM = 1, ROW_SILU = 2, ROW_PLAIN = 3 };

struct RowArgs {
    const void* in; const void* weight; void* residual;      // in: [rows, cols] (ROW_SILU: [rows, 2*cols])
    int64_t in_stride;                                       // elements between rows of `in`
    void* out; int8_t* codes; float* scale;                  // one of out / codes
    int nvec;                                                // cols / 8
    float eps, inv_cols;
    int64_t rows;
};

// silu(g) * u.  1 + exp(-g) reaches 2^128 before it overflows, and its reciprocal is subnormal from 2^126 on, where g / (1 + exp(-g)) is
// still a normal number: both are taken 2^16 apart, which is given back by u (exactly: a 16-bit number times 2^-16 is an fp32 number).
__device__ __forceinline__ float silu_mul(float g, float u) {
    constexpr float kDown = 1.f / 65536.f;
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(ptx::ex2(g * -1.4426950408889634f), kDown, kDown)));
    return g * (r * (u * kDown));
}

template <int VPT> struct RowData { uint4 a[VPT], b[VPT]; };

// nt threads share a row: a warp (WARP) or the CTA
template <typename T, int MODE, int VPT, bool QUANT, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : (VPT == 2 ? 512 : (VPT == 4 ? 512 : 1024))) row_kernel(RowArgs a) {
    constexpr bool kNorm = MODE == ROW_ADD_NORM || MODE == ROW_NORM;
    const int lane = threadIdx.x & 31;
    const int tid = WARP ? lane : threadIdx.x, nt = WARP ? 32 : blockDim.x;
    const int64_t first = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    const int64_t step = WARP ? (int64_t)gridDim.x * (blockDim.x >> 5) : a.rows;      // a CTA takes one row
    if (QUANT) grid_dependents_launch();              // a product of the codes is what comes next
    const uint4* wv = reinterpret_cast<const uint4*>(a.weight);
    __shared__ float s_ss[32];
    __shared__ uint32_t s_mx[32];

    auto load = [&](int64_t row, RowData<VPT>& d) {
        const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.in) + row * a.in_stride);
        const uint4* res = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.residual) + row * (int64_t)a.nvec * 8);
#pragma unroll
        for (int c = 0; c < VPT; ++c) {
            const int i = tid + c * nt;
            if (i < a.nvec) {
                d.a[c] = src[i];
                if (MODE == ROW_ADD_NORM) d.b[c] = res[i];
                if (MODE == ROW_SILU) d.b[c] = src[a.nvec + i];
            }
        }
    };
    RowData<VPT> d;
    if (first < a.rows) load(first, d);
#pragma unroll 1
    for (int64_t row = first; row < a.rows; row += step) {
        float t[VPT][8];
        float ss = 0.f;
        uint32_t amax = 0;
        uint4* res = MODE == ROW_ADD_NORM ? reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.residual) + row * (int64_t)a.nvec * 8) : nullptr;
#pragma unroll
        for (int c = 0; c < VPT; ++c) {
            const int i = tid + c * nt;
            if (i < a.nvec) {
                const uint32_t u[4] = {d.a[c].x, d.a[c].y, d.a[c].z, d.a[c].w}, q[4] = {d.b[c].x, d.b[c].y, d.b[c].z, d.b[c].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float2 f = Cvt<T>::to_f2(u[k]);
                    if (MODE == ROW_ADD_NORM) { const float2 g = Cvt<T>::to_f2(q[k]); f.x += g.x; f.y += g.y; }
                    if (MODE == ROW_SILU) {
                        const float2 g = Cvt<T>::to_f2(q[k]);
                        f.x = silu_mul(f.x, g.x);
                        f.y = silu_mul(f.y, g.y);
                    }
                    if (kNorm) { ss = fmaf(f.x, f.x, ss); ss = fmaf(f.y, f.y, ss); }
                    t[c][2 * k] = f.x; t[c][2 * k + 1] = f.y;
                }
                if (MODE == ROW_ADD_NORM)
                    res[i] = make_uint4(Cvt<T>::pack(t[c][0], t[c][1]), Cvt<T>::pack(t[c][2], t[c][3]), Cvt<T>::pack(t[c][4], t[c][5]), Cvt<T>::pack(t[c][6], t[c][7]));
            }
        }
        if (WARP && row + step < a.rows) load(row + step, d);
#pragma unroll
        for (int c = 0; c < VPT; ++c) {
            const int i = tid + c * nt;
            if (i < a.nvec) {
                if (kNorm) {
                    const uint4 w = __ldg(wv + i);
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
        if (kNorm) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        }
        if (QUANT) amax = __reduce_max_sync(0xffffffffu, amax);
        if (!WARP) {
            const int warps = nt >> 5;
            if (lane == 0) { s_ss[threadIdx.x >> 5] = ss; s_mx[threadIdx.x >> 5] = amax; }
            __syncthreads();
            ss = 0.f; amax = 0;
            for (int i = 0; i < warps; ++i) { ss += s_ss[i]; amax = max(amax, s_mx[i]); }
        }
        const float rstd = kNorm ? rsqrtf(fmaf(ss, a.inv_cols, a.eps)) : 1.f;
        if (QUANT) {
            // the maximum of |t * w * rstd| is that of |t * w| times rstd: rounding a product is monotonic
            const RowScale r = row_scale(abs_bits(__uint_as_float(amax) * rstd), kInt8Top);
            if (tid == 0) a.scale[row] = r.scale;
            uint2* dst = reinterpret_cast<uint2*>(a.codes + row * (int64_t)a.nvec * 8);
#pragma unroll
            for (int c = 0; c < VPT; ++c) {
                const int i = tid + c * nt;
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
                const int i = tid + c * nt;
                if (i < a.nvec) {
                    uint32_t o[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) o[k] = Cvt<T>::pack(t[c][2 * k] * rstd, t[c][2 * k + 1] * rstd);
                    dst[i] = make_uint4(o[0], o[1], o[2], o[3]);
                }
            }
        }
    }
}

// eight codes per lane and step, four steps in flight
template <typename OT>
__global__ void __launch_bounds__(256) dequantize_rows_kernel(OT* __restrict__ out, const int8_t* __restrict__ codes,
                                                              const float* __restrict__ scale, int64_t rows, int vecs) {
    constexpr int U = 4;
    const int64_t total = rows * vecs, stride = (int64_t)gridDim.x * 256;
    for (int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x; i0 < total; i0 += U * stride) {
        uint2 w[U];
        float s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = i0 + u * stride;
            if (i < total) {
                w[u] = __ldcs(reinterpret_cast<const uint2*>(codes) + i);
                s[u] = scale[i / vecs];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = i0 + u * stride;
            if (i >= total) continue;
            float lo[4], hi[4], f[8];
            unpack_codes4<ESP_CODE_INT8>(w[u].x, lo);
            unpack_codes4<ESP_CODE_INT8>(w[u].y, hi);
#pragma unroll
            for (int k = 0; k < 4; ++k) { f[k] = lo[k] * s[u]; f[4 + k] = hi[k] * s[u]; }
            if constexpr (sizeof(OT) == 4) {
                float4* o = reinterpret_cast<float4*>(out + i * 8);
                o[0] = make_float4(f[0], f[1], f[2], f[3]);
                o[1] = make_float4(f[4], f[5], f[6], f[7]);
            } else {
                *reinterpret_cast<uint4*>(out + i * 8) = make_uint4(Cvt<OT>::pack(f[0], f[1]), Cvt<OT>::pack(f[2], f[3]),
                                                                    Cvt<OT>::pack(f[4], f[5]), Cvt<OT>::pack(f[6], f[7]));
            }
        }
    }
}

constexpr int kMaxRowCols = 8 * 8 * 1024;          // VPT 8 x 1024 threads x 8 elements

template <typename T, int MODE, bool QUANT>
static int launch_row(RowArgs a, int64_t rows, int cols, cudaStream_t s) {
    a.nvec = cols / 8;
    a.inv_cols = 1.f / (float)cols;
    a.rows = rows;
    if (a.nvec <= 64) {
        const int64_t want = (rows + 7) / 8, cap = kNumSMs * 16;
        const unsigned grid = (unsigned)(want < cap ? want : cap);
        if (a.nvec <= 32) row_kernel<T, MODE, 1, QUANT, true><<<grid, 256, 0, s>>>(a);
        else row_kernel<T, MODE, 2, QUANT, true><<<grid, 256, 0, s>>>(a);
    } else {
        // 16-byte vectors per thread: 2 keeps a row of 4096 in 256 threads; wider rows hold more per thread up to 8
        const int vpt = a.nvec <= 2 * 512 ? 2 : (a.nvec <= 4 * 512 ? 4 : 8);
        const int nt = ((a.nvec + vpt - 1) / vpt + 31) / 32 * 32;
        const unsigned grid = (unsigned)rows;
        if (vpt == 2) row_kernel<T, MODE, 2, QUANT, false><<<grid, nt, 0, s>>>(a);
        else if (vpt == 4) row_kernel<T, MODE, 4, QUANT, false><<<grid, nt, 0, s>>>(a);
        else row_kernel<T, MODE, 8, QUANT, false><<<grid, nt, 0, s>>>(a);
    }
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
    RowArgs a{in, weight, residual, hidden, out, nullptr, nullptr, 0, eps, 0.f, 0};
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
    RowArgs a{in, weight, residual, hidden, nullptr, codes, scale, 0, eps, 0.f, 0};
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
    RowArgs a{io, nullptr, nullptr, 2 * (int64_t)ffn_inter_dim, nullptr, codes, scale, 0, 0.f, 0.f, 0};
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
    RowArgs a{x, nullptr, nullptr, x_row_stride, nullptr, codes, scale, 0, 0.f, 0.f, 0};
    return dtype == ESP_DTYPE_F16 ? launch_row<__half, ROW_PLAIN, true>(a, rows, cols, (cudaStream_t)stream)
                                  : launch_row<__nv_bfloat16, ROW_PLAIN, true>(a, rows, cols, (cudaStream_t)stream);
}

extern "C" int esp_dequantize_rows(void* out, const int8_t* codes, const float* scale, int64_t rows, int32_t cols, int32_t dtype, void* stream) {
    if (rows == 0) return ESP_OK;
    if (!out || !codes || !scale || rows < 0 || cols <= 0) return ESP_ERR_BAD_ARG;
    if (cols % 8 || !aligned16(out) || ((uintptr_t)codes & 7u)) return ESP_ERR_ALIGNMENT;
    const int64_t want = (rows * (cols / 8) + 1023) / 1024, cap = (int64_t)kNumSMs * 32;
    const unsigned grid = (unsigned)(want < cap ? want : cap);
    cudaStream_t s = (cudaStream_t)stream;
#define ESP_DQ(OT) dequantize_rows_kernel<OT><<<grid, 256, 0, s>>>((OT*)out, codes, scale, rows, cols / 8);
    if (dtype == ESP_DTYPE_F16) ESP_DQ(__half)
    else if (dtype == ESP_DTYPE_BF16) ESP_DQ(__nv_bfloat16)
    else if (dtype == ESP_DTYPE_F32) ESP_DQ(float)
    else return ESP_ERR_BAD_ARG;
#undef ESP_DQ
    ESP_LAUNCH_CHECK("dequantize_rows_kernel");
    return ESP_OK;
}
