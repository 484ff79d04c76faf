// Split-KV decode attention over a KV pool held in 8 bits (codes and one fp32 scale per slot and head, quant_common.cuh):
//   s_t = (q . ck_t) * k_scale_t * sm_scale,   p_t = exp(s_t - m),   o = sum_t p_t * v_scale_t * cv_t / sum_t p_t
// Same splits, partials and merge as the 16-bit form (decode_attention.cu).
//
// Bound by HBM: 2 * (128 + 4) bytes per token and kv head, each read once.  At that rate one SM has to take in a code every
// 1/23 of a cycle and multiply it with up to 8 query heads, which is past what fp32 lanes do next to the conversion; so codes
// become f16 (exactly: 8 bits fit) and the products run on the tensor cores (mma.sync m16n8k16, fp32 sums), which are far
// from their limit here.  No shared memory and no shuffles of data: each lane loads 16-byte pieces straight from global
// memory and its pieces ARE operand fragments, because the order of the summed index (head dims for S, tokens for O) is free:
//   S [heads 16 x tokens 8] = Q K^T   B fragment of lane (g, c): token g, dims {16c..16c+15, 64+16c..64+16c+15}, one word of
//                                     four codes per MMA; Q fragments are loaded once in the same dim order.
//   O^T [dims 16 x heads 8] += V^T P^T  A fragment of lane (g, c): dims 16g..16g+15, tokens 2c, 2c+1, 2c+8, 2c+9 (words of two
//                                     tokens interleaved byte by byte); P^T's fragment is what the lane holds of S.
// (lane = 4g + c.)  A warp takes 16 tokens per step, the next step's loads are in flight meanwhile.
//
// Precision.  q is scaled by a power of two per head so that its largest element is near 2^7 in f16: exact down to 2^-21 of
// it.  Scores, maxima, sums and outputs are fp32.  The weights p * v_scale are rounded to f16 (11 bits) before the second
// product, relative to 2^-8 * the largest v_scale seen by the warp: like the 16-bit P of the prefill kernels, one rounding of
// 2^-12 relative per term.
#include "quant_common.cuh"
#include "sm100_ptx.cuh"

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
    float scale_log2; int64_t pool_rows; int head_tiles;
};

constexpr int kQ8Warps = 4, kQ8HeadTile = 8;

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Four codes of a word as two f16 pairs: codes 0, 1 and codes 2, 3.  int8: code + 128 placed under the exponent of 1024 is
// 1152 + code exactly, from which 1152 is taken away.
template <int CODE>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (CODE == ESP_CODE_INT8) {
        const uint32_t u = w ^ 0x80808080u;
        const __half2 k = __half2half2(__ushort_as_half(0x6480));        // 1152
        uint32_t l = __byte_perm(u, 0x64646464u, 0x4140), h = __byte_perm(u, 0x64646464u, 0x4342);
        __half2 x = __hsub2(*reinterpret_cast<__half2*>(&l), k), y = __hsub2(*reinterpret_cast<__half2*>(&h), k);
        lo = *reinterpret_cast<uint32_t*>(&x); hi = *reinterpret_cast<uint32_t*>(&y);
    } else {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(lo), "=r"(hi) : "r"(w));
    }
}

// A warp's steps (16 tokens of one kv head each) pass through a ring in shared memory, filled with 16-byte asynchronous copies.
// Every lane reads back exactly the bytes it copied, so the ring is a register file that does not hold registers while the
// copies are under way; only the scales and the mask of present tokens pass between lanes.
constexpr int kQ8Stages = 4;
struct StepQ8 {
    uint4 kv[8][32];        // [piece][lane]: K tokens g, g + 8 x dims (16c.., 64 + 16c..), V tokens 2c, 2c + 1, 2c + 8, 2c + 9 x dims 16g..
    float k_scale[16], v_scale[16];
};
struct SmemQ8 {
    StepQ8 ring[kQ8Warps][kQ8Stages];
    uint32_t present[kQ8Warps][kQ8Stages];      // bit t: token t of the step exists
};
struct MergeQ8 {                                // over the ring, once it is used up
    float o[kQ8Warps][kQ8HeadTile][132];
    float m[kQ8Warps][kQ8HeadTile], l[kQ8Warps][kQ8HeadTile], v[kQ8Warps];
};
static_assert(sizeof(MergeQ8) <= sizeof(SmemQ8), "the merge reuses the ring");

// copies `bytes` (16 or, for a token that does not exist, 0: the rest is filled with zeros)
__device__ __forceinline__ void cp_async16(void* dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(void* dst, const void* src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(ptx::smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}

template <typename T, int CODE>
__global__ void __launch_bounds__(kQ8Warps * 32, 3) decode_stage1_q8_kernel(DecodeQ8Args a) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    SmemQ8& sm = *reinterpret_cast<SmemQ8*>(smem_raw);
    // all kv heads of a split run next to each other: their rows and their scales (eight heads to a 32-byte sector) are neighbours
    const int blk = blockIdx.x / a.head_tiles, ht = blockIdx.x - blk * a.head_tiles, b = blockIdx.y;
    const int len = a.b_seqlen[b];
    const int t0 = blk * a.seq_block_size;
    int t1 = min(t0 + a.seq_block_size, len);
    if (t1 <= t0) return;
    const int tiles_per_kv = (a.group + kQ8HeadTile - 1) / kQ8HeadTile;
    const int kvh = ht / tiles_per_kv, hsub = ht - kvh * tiles_per_kv;
    const int h0 = kvh * a.group + hsub * kQ8HeadTile;
    const int nheads = min(kQ8HeadTile, a.group - hsub * kQ8HeadTile);
    const int req = a.b_req_idx[b];
    if (req < 0 || req >= a.rtt_rows || len > a.rtt_cols) {
        if (threadIdx.x == 0) q8_report(1, req);
        t1 = t0;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;

    // tokens [w0, w1) of this warp, whole groups of 32 except at the end
    const int per_warp = ((t1 - t0 + kQ8Warps * 32 - 1) / (kQ8Warps * 32)) * 32;
    const int w0 = min(t0 + warp * per_warp, t1), w1 = min(w0 + per_warp, t1);
    const int32_t* rtt = a.req_to_tokens + (w1 > w0 ? (int64_t)req * a.rtt_stride : 0);
    const uint8_t* kbase = a.k + (int64_t)kvh * a.k_stride_h + c * 16;
    const uint8_t* vbase = a.v + (int64_t)kvh * a.v_stride_h + g * 16;
    const float* sbase = lane < 16 ? a.k_scale + kvh : a.v_scale + kvh;
    const int64_t s_stride = lane < 16 ? a.ks_stride_t : a.vs_stride_t;

    // slots of 32 tokens, one per lane; -1: no such token
    auto load_slots = [&](int t) -> int {
        if (t + lane >= w1) return -1;
        const int s = rtt[t + lane];
        if (s < 0 || s >= a.pool_rows) { q8_report(0, s); return -1; }
        return s;
    };
    // copies step `half` of the group of 32 tokens whose slots the lanes hold; a token that does not exist (its address would
    // be that of slot 0, which is there) is filled with zeros
    auto issue = [&](int stage, int group_slots, int half) {
        StepQ8& d = sm.ring[warp][stage];
        const int mine = __shfl_sync(0xffffffffu, group_slots, half * 16 + (lane & 15));
        const uint32_t present = __ballot_sync(0xffffffffu, mine >= 0) & 0xffffu;
        if (lane == 0) sm.present[warp][stage] = present;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int s = __shfl_sync(0xffffffffu, mine, g + 8 * i);
            const uint8_t* p = kbase + (int64_t)max(s, 0) * a.k_stride_t;
            cp_async16(&d.kv[2 * i][lane], p, s >= 0 ? 16 : 0);
            cp_async16(&d.kv[2 * i + 1][lane], p + 64, s >= 0 ? 16 : 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = __shfl_sync(0xffffffffu, mine, 2 * c + (i & 1) + 8 * (i >> 1));
            cp_async16(&d.kv[4 + i][lane], vbase + (int64_t)max(s, 0) * a.v_stride_t, s >= 0 ? 16 : 0);
        }
        cp_async4(lane < 16 ? &d.k_scale[lane] : &d.v_scale[lane - 16], sbase + (int64_t)max(mine, 0) * s_stride, mine >= 0 ? 4 : 0);
    };

    // the next step to copy: step n_issue of the warp, from group n_issue / 2
    const int steps = (w1 - w0 + 15) >> 4;
    int n_issue = 0, slots = load_slots(w0), slots_next = load_slots(w0 + 32);
    auto issue_next = [&](int stage) {
        if (n_issue < steps) {
            issue(stage, slots, n_issue & 1);
            if (n_issue & 1) { slots = slots_next; slots_next = load_slots(w0 + (n_issue + 1) * 16 + 32); }
            ++n_issue;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");             // an empty group keeps the count
    };
#pragma unroll
    for (int i = 0; i < kQ8Stages - 1; ++i) issue_next(i);

    // Q fragments: row g is head g of the tile (rows 8-15 of the MMA stay zero), dims in the order of the K words
    uint32_t qf[8][2];
    float qs;
    {
        float x[32], amax = 0.f;
        const T* qp = reinterpret_cast<const T*>(a.q) + ((int64_t)b * a.num_q_heads + h0 + g) * 128 + c * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 u = g < nheads ? *reinterpret_cast<const uint4*>(qp + (i >> 1) * 64 + (i & 1) * 8) : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = Cvt<T>::to_f2(w[j]);
                x[8 * i + 2 * j] = f.x; x[8 * i + 2 * j + 1] = f.y;
                amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // 2^(7 - e) with 2^e <= amax; e held in [-100, 126] so that both powers are normal numbers
        int e = (int)(__float_as_uint(amax) >> 23) - 127;
        e = min(max(e, -100), 126);
        const float up = __uint_as_float((uint32_t)(127 + 7 - e) << 23);
        qs = a.scale_log2 * __uint_as_float((uint32_t)(127 - 7 + e) << 23);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            qf[j][0] = Cvt<__half>::pack(x[4 * j] * up, x[4 * j + 1] * up);
            qf[j][1] = Cvt<__half>::pack(x[4 * j + 2] * up, x[4 * j + 3] * up);
        }
    }

    float acc[8][4] = {};                 // MMA j: dims 16g + 2j (0, 1) and 16g + 2j + 1 (2, 3) of heads 2c, 2c + 1
    float m_ref = -INFINITY, l_run = 0.f; // of head g; l over this lane's tokens only
    float v_ref = 0.f, v_mul = 0.f;       // weights are held as p * v_scale * v_mul, v_mul = 2^12 / v_ref, v_ref >= every v_scale so far

    auto compute = [&](const StepQ8& d, uint32_t present) {
        float s[2][4] = {};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 x = d.kv[2 * i][lane], y = d.kv[2 * i + 1][lane];
            const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint32_t lo, hi;
                codes_to_f16<CODE>(w[j], lo, hi);
                mma_f16(s[i], qf[j][0], 0u, qf[j][1], 0u, lo, hi);
            }
        }
        float sc[4], vs[4];               // of tokens 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 kf = *reinterpret_cast<const float2*>(&d.k_scale[2 * c + 8 * i]);
            const float2 vf = *reinterpret_cast<const float2*>(&d.v_scale[2 * c + 8 * i]);
            sc[2 * i] = s[i][0] * (kf.x * qs); sc[2 * i + 1] = s[i][1] * (kf.y * qs);
            vs[2 * i] = vf.x; vs[2 * i + 1] = vf.y;
        }
        if (present != 0xffffu) {         // zeros were copied for the others: only their scores need a word
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!((present >> (2 * c + (i & 1) + 8 * (i >> 1))) & 1u)) sc[i] = -INFINITY;
        }
        float smax = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
        const float vmax = fmaxf(fmaxf(fabsf(vs[0]), fabsf(vs[1])), fmaxf(fabsf(vs[2]), fabsf(vs[3])));
        // both references move rarely: the maximum only once a score is 3 above it (p stays below 2^3, weights below 2^15)
        if (__any_sync(0xffffffffu, smax > m_ref + 3.f || vmax > v_ref)) {
            smax = fmaxf(smax, __shfl_xor_sync(0xffffffffu, smax, 1));
            smax = fmaxf(smax, __shfl_xor_sync(0xffffffffu, smax, 2));
            float vm = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 1));
            vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, 2));
            const float m_new = fmaxf(m_ref, smax);
            float alpha = m_new == m_ref ? 1.f : exp2f(m_ref - m_new);
            m_ref = m_new;
            l_run *= alpha;
            if (vm > v_ref) {             // the same in every lane
                const float v_new = fmaxf(4.f * vm, 1e-34f);
                alpha *= v_ref / v_new;
                v_ref = v_new; v_mul = 4096.f / v_new;
            }
            const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * c), a1 = __shfl_sync(0xffffffffu, alpha, 8 * c + 4);
#pragma unroll
            for (int j = 0; j < 8; ++j) { acc[j][0] *= a0; acc[j][1] *= a1; acc[j][2] *= a0; acc[j][3] *= a1; }
        }
        const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
        float wgt[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p = ptx::ex2(sc[i] - m_use);
            l_run += p;
            wgt[i] = p * (vs[i] * v_mul);
        }
        const uint32_t b0 = Cvt<__half>::pack(wgt[0], wgt[1]), b1 = Cvt<__half>::pack(wgt[2], wgt[3]);
        uint32_t vw[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) { const uint4 x = d.kv[4 + i][lane]; vw[i][0] = x.x; vw[i][1] = x.y; vw[i][2] = x.z; vw[i][3] = x.w; }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {                      // dims 4w + 2h, 4w + 2h + 1 of this lane's 16
                const uint32_t sel = h ? 0x7362 : 0x5140;
                uint32_t x0, x1, y0, y1;
                codes_to_f16<CODE>(__byte_perm(vw[0][w], vw[1][w], sel), x0, x1);
                codes_to_f16<CODE>(__byte_perm(vw[2][w], vw[3][w], sel), y0, y1);
                mma_f16(acc[2 * w + h], x0, x1, y0, y1, b0, b1);
            }
        }
    };

    int stage = 0;
#pragma unroll 1
    for (int i = 0; i < steps; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kQ8Stages - 2) : "memory");
        __syncwarp();                     // the other lanes' scales and the mask are there; all have left the stage filled next
        issue_next(stage == 0 ? kQ8Stages - 1 : stage - 1);
        compute(sm.ring[warp][stage], sm.present[warp][stage]);
        stage = stage + 1 == kQ8Stages ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();

    // the four warps' states: heads of this tile, in units of each warp's own reference
    MergeQ8& mg = *reinterpret_cast<MergeQ8*>(smem_raw);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
    if (c == 0) { mg.m[warp][g] = m_ref; mg.l[warp][g] = l_run; }
    if (lane == 0) mg.v[warp] = v_ref * (1.f / 4096.f);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        *reinterpret_cast<float2*>(&mg.o[warp][2 * c][16 * g + 2 * j]) = make_float2(acc[j][0], acc[j][2]);
        *reinterpret_cast<float2*>(&mg.o[warp][2 * c + 1][16 * g + 2 * j]) = make_float2(acc[j][1], acc[j][3]);
    }
    __syncthreads();
    const int d = threadIdx.x;
    for (int h = 0; h < nheads; ++h) {
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kQ8Warps; ++w) M = fmaxf(M, mg.m[w][h]);
        const float Mu = M == -INFINITY ? 0.f : M;
        float L = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < kQ8Warps; ++w) {
            const float f = exp2f(mg.m[w][h] - Mu);             // 0 for a warp that saw no token
            L += mg.l[w][h] * f;
            o += mg.o[w][h][d] * (f * mg.v[w]);
        }
        const int64_t row = ((int64_t)blk * a.batch + b) * a.num_q_heads + h0 + h;
        a.mid_o[row * 128 + d] = L == 0.f ? 0.f : o / L;
        if (d == 0) a.mid_lse[row] = L == 0.f ? -INFINITY : (Mu + log2f(L)) * kLn2Q8;
    }
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
                   (sm_scale > 0.f ? sm_scale : 1.0f / sqrtf((float)head_dim)) * kLog2eQ8, pool_rows, 0};
    a.head_tiles = num_kv_heads * ((a.group + kQ8HeadTile - 1) / kQ8HeadTile);
    const int64_t nblk = (max_len_in_batch + (int64_t)seq_block_size - 1) / seq_block_size;
    if (nblk * a.head_tiles > 2147483647LL || nblk * seq_block_size > 2147483647LL) return ESP_ERR_TOO_LARGE;
    const dim3 grid((unsigned)(nblk * a.head_tiles), batch);
    cudaStream_t s = (cudaStream_t)stream;
#define ESP_S1Q(T, C)                                                                                                             \
    {                                                                                                                            \
        ESP_CUDA_TRY(cudaFuncSetAttribute(decode_stage1_q8_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(SmemQ8))); \
        decode_stage1_q8_kernel<T, C><<<grid, kQ8Warps * 32, sizeof(SmemQ8), s>>>(a);                                              \
    }
    if (dtype == ESP_DTYPE_F16) {
        if (code == ESP_CODE_INT8) ESP_S1Q(__half, ESP_CODE_INT8) else ESP_S1Q(__half, ESP_CODE_E4M3)
    } else {
        if (code == ESP_CODE_INT8) ESP_S1Q(__nv_bfloat16, ESP_CODE_INT8) else ESP_S1Q(__nv_bfloat16, ESP_CODE_E4M3)
    }
#undef ESP_S1Q
    ESP_LAUNCH_CHECK("decode_stage1_q8_kernel");
    return ESP_OK;
}
