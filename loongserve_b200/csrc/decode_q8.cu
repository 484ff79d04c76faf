// Split-KV decode attention over a KV pool held in 8 bits (codes and one fp32 scale per slot and head, quant_common.cuh):
//   s_t = (q . ck_t) * k_scale_t * sm_scale,   p_t = exp(s_t - m),   o = sum_t p_t * v_scale_t * cv_t / sum_t p_t
// Same splits, partials and merge as the 16-bit form (decode_attention.cu).
//
// First form: eight lanes share a 128-byte code row, fp32 arithmetic.
#include "quant_common.cuh"

namespace esp {

constexpr float kLog2eQ8 = 1.4426950408889634f, kLn2Q8 = 0.6931471805599453f;

// {ESP_ERR_BAD_SLOT, block, 0 slot id / 1 request row, value}, as in the 16-bit kernels
__device__ int g_decode_q8_status[4];

__device__ __noinline__ void q8_report(int which, int value) {
    if (atomicCAS(&g_decode_q8_status[0], 0, ESP_ERR_BAD_SLOT) == 0) {
        g_decode_q8_status[1] = blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z);
        g_decode_q8_status[2] = which;
        g_decode_q8_status[3] = value;
    }
}

struct DecodeQ8Args {
    float* mid_o; float* mid_lse; const void* q; const uint8_t* k; const uint8_t* v; const float* k_scale; const float* v_scale;
    int64_t k_stride_t, k_stride_h, v_stride_t, v_stride_h, ks_stride_t, vs_stride_t;
    const int32_t* req_to_tokens; int64_t rtt_stride; int rtt_rows, rtt_cols;
    const int32_t *b_req_idx, *b_seqlen;
    int batch, num_q_heads, num_kv_heads, group, seq_block_size;
    float scale_log2; int64_t pool_rows;
};

template <typename T, int CODE>
__global__ void __launch_bounds__(128) decode_stage1_q8_kernel(DecodeQ8Args a) {
    const int blk = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int len = a.b_seqlen[b];
    const int t0 = blk * a.seq_block_size;
    int t1 = min(t0 + a.seq_block_size, len);
    if (t1 <= t0) return;
    const int req = a.b_req_idx[b];
    bool row_ok = req >= 0 && req < a.rtt_rows && len <= a.rtt_cols;
    if (!row_ok) { if (threadIdx.x == 0) q8_report(1, req); t1 = t0; }
    const int32_t* rtt = a.req_to_tokens + (row_ok ? (int64_t)req * a.rtt_stride : 0);
    const int kvh = h / a.group;
    const int grp = threadIdx.x >> 3, lane8 = threadIdx.x & 7;
    float qf[16], acc[16] = {}, m_run = -INFINITY, l_run = 0.f;
    {
        const T* qp = reinterpret_cast<const T*>(a.q) + ((int64_t)b * a.num_q_heads + h) * 128 + lane8 * 16;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 f = Cvt<T>::to_f2(reinterpret_cast<const uint32_t*>(qp)[i]);
            qf[2 * i] = f.x * a.scale_log2; qf[2 * i + 1] = f.y * a.scale_log2;
        }
    }
    for (int base = t0; base < t1; base += 16) {
        const int t = base + grp;
        int64_t slot = t < t1 ? rtt[t] : -1;
        if (t < t1 && (slot < 0 || slot >= a.pool_rows)) { if (lane8 == 0) q8_report(0, (int)slot); slot = -1; }
        uint4 kc = make_uint4(0, 0, 0, 0), vc = kc;
        float ks = 0.f, vs = 0.f;
        if (slot >= 0) {
            kc = ld_nc_v4(a.k + slot * a.k_stride_t + (int64_t)kvh * a.k_stride_h + lane8 * 16);
            vc = ld_nc_v4(a.v + slot * a.v_stride_t + (int64_t)kvh * a.v_stride_h + lane8 * 16);
            ks = a.k_scale[slot * a.ks_stride_t + kvh]; vs = a.v_scale[slot * a.vs_stride_t + kvh];
        }
        const uint32_t kw[4] = {kc.x, kc.y, kc.z, kc.w}, vw[4] = {vc.x, vc.y, vc.z, vc.w};
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float f[4];
            unpack_codes4<CODE>(kw[j], f);
#pragma unroll
            for (int i = 0; i < 4; ++i) s = fmaf(qf[4 * j + i], f[i], s);
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s = slot >= 0 ? s * ks : -INFINITY;
        const float m_new = fmaxf(m_run, s), m_use = m_new == -INFINITY ? 0.f : m_new;
        const float al = exp2f(m_run - m_use), p = exp2f(s - m_use);
        l_run = l_run * al + p;
        m_run = m_new;
        const float w = slot >= 0 ? p * vs : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float f[4];
            unpack_codes4<CODE>(vw[j], f);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[4 * j + i] = fmaf(w, f[i], acc[4 * j + i] * al);
        }
    }
    __shared__ float s_acc[16][128], s_m[16], s_l[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) s_acc[grp][lane8 * 16 + i] = acc[i];
    if (lane8 == 0) { s_m[grp] = m_run; s_l[grp] = l_run; }
    __syncthreads();
    float M = -INFINITY;
    for (int i = 0; i < 16; ++i) M = fmaxf(M, s_m[i]);
    const float Mu = M == -INFINITY ? 0.f : M;
    float L = 0.f, o = 0.f;
    for (int i = 0; i < 16; ++i) { const float w = exp2f(s_m[i] - Mu); L += s_l[i] * w; o += s_acc[i][threadIdx.x] * w; }
    const int64_t row = ((int64_t)blk * a.batch + b) * a.num_q_heads + h;
    a.mid_o[row * 128 + threadIdx.x] = L == 0.f ? 0.f : o / L;
    if (threadIdx.x == 0) a.mid_lse[row] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2Q8;
}

int decode_q8_status(int32_t out[4], int32_t clear) {
    ESP_CUDA_TRY(cudaMemcpyFromSymbol(out, g_decode_q8_status, sizeof(int) * 4));
    if (clear) {
        int zero[4] = {0, 0, 0, 0};
        ESP_CUDA_TRY(cudaMemcpyToSymbol(g_decode_q8_status, zero, sizeof(zero)));
    }
    return ESP_OK;
}

}  // namespace esp

using namespace esp;

extern "C" int esp_decode_stage1_q8(float* mid_o, float* mid_lse, const void* q, const void* k, const void* v, const float* k_scale,
                                    const float* v_scale, int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h,
                                    int64_t k_scale_stride_t, int64_t v_scale_stride_t, const int32_t* req_to_tokens,
                                    int64_t req_to_tokens_stride, int32_t req_rows, int32_t req_cols, const int32_t* b_req_idx,
                                    const int32_t* b_seqlen, int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                    int32_t max_len_in_batch, int32_t seq_block_size, int32_t dtype, int32_t code, float sm_scale,
                                    int64_t pool_rows, void* stream) {
    if (batch == 0 || max_len_in_batch <= 0) return ESP_OK;
    if (!mid_o || !mid_lse || !q || !k || !v || !k_scale || !v_scale || !req_to_tokens || !b_req_idx || !b_seqlen || batch < 0 ||
        num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads || seq_block_size <= 0 || req_rows <= 0 || req_cols <= 0 ||
        pool_rows <= 0)
        return ESP_ERR_BAD_ARG;
    if (dtype != ESP_DTYPE_F16 && dtype != ESP_DTYPE_BF16) return ESP_ERR_BAD_ARG;
    if (code != ESP_CODE_INT8 && code != ESP_CODE_E4M3) return ESP_ERR_BAD_ARG;
    if (head_dim != 128) return ESP_ERR_UNSUPPORTED;
    if (batch > 65535 || num_q_heads > 65535) return ESP_ERR_TOO_LARGE;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || k_stride_t % 16 || k_stride_h % 16 || v_stride_t % 16 || v_stride_h % 16 ||
        ((uintptr_t)k_scale & 3u) || ((uintptr_t)v_scale & 3u))
        return ESP_ERR_ALIGNMENT;
    DecodeQ8Args a{mid_o, mid_lse, q, (const uint8_t*)k, (const uint8_t*)v, k_scale, v_scale, k_stride_t, k_stride_h, v_stride_t, v_stride_h,
                   k_scale_stride_t, v_scale_stride_t, req_to_tokens, req_to_tokens_stride, req_rows, req_cols, b_req_idx, b_seqlen, batch,
                   num_q_heads, num_kv_heads, num_q_heads / num_kv_heads, seq_block_size,
                   (sm_scale > 0.f ? sm_scale : 1.0f / sqrtf((float)head_dim)) * kLog2eQ8, pool_rows};
    const dim3 grid((unsigned)((max_len_in_batch + (int64_t)seq_block_size - 1) / seq_block_size), num_q_heads, batch);
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == ESP_DTYPE_F16) {
        if (code == ESP_CODE_INT8) decode_stage1_q8_kernel<__half, ESP_CODE_INT8><<<grid, 128, 0, s>>>(a);
        else decode_stage1_q8_kernel<__half, ESP_CODE_E4M3><<<grid, 128, 0, s>>>(a);
    } else {
        if (code == ESP_CODE_INT8) decode_stage1_q8_kernel<__nv_bfloat16, ESP_CODE_INT8><<<grid, 128, 0, s>>>(a);
        else decode_stage1_q8_kernel<__nv_bfloat16, ESP_CODE_E4M3><<<grid, 128, 0, s>>>(a);
    }
    ESP_LAUNCH_CHECK("decode_stage1_q8_kernel");
    return ESP_OK;
}
