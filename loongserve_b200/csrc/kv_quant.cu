// The KV pool in 8 bits: rows are quantised as they are written to their slots, and read back from them.
//
// A pool row keeps, per head, head_dim codes and one fp32 scale (quant_common.cuh).  The scale belongs to ONE token and head:
// slots are handed out token by token, so tokens of different requests may be neighbours and a scale over several slots
// would have to be revised by every later write.
//
// HBM bound.  Per head row of D: write reads 2*D and stores D + 4 bytes, read-back the other way round.  Writing, LPR lanes share a
// head row with 16 elements each: two 16-byte loads, the row's maximum by shuffles over its lanes, a 16-byte store of codes; the
// data is read once and stays in registers.  A lane group's token and head come from shifts, not from a division of the row
// number: with the division, and with 8 elements per lane, the instructions were the bound (16384 tokens x 64 heads: 82 and
// 108 us; as it is 71 us for 407 MB, the way back 68).  The keep-range form has one row of a lane group in flight and takes 82 us for the same
// rows from 8 requests.
#include "quant_common.cuh"

namespace esp {

// Like the 16-bit pool kernels: a slot id outside the pool is never dereferenced; the first one is recorded as
// {ESP_ERR_BAD_SLOT, kernel id, position, id clamped to int32}.
__device__ int g_kv_q8_status[4];

__device__ __forceinline__ bool q8_slot_ok(int64_t slot, int64_t pool_rows, int kernel_id, int64_t pos) {
    if (slot >= 0 && slot < pool_rows) return true;
    if (atomicCAS(&g_kv_q8_status[0], 0, ESP_ERR_BAD_SLOT) == 0) {
        g_kv_q8_status[1] = kernel_id;
        g_kv_q8_status[2] = (int)(pos > 2147483647LL ? 2147483647LL : pos);
        g_kv_q8_status[3] = (int)(slot > 2147483647LL ? 2147483647LL : (slot < -2147483647LL ? -2147483647LL : slot));
    }
    return false;
}

__device__ __forceinline__ int64_t idx_at(const void* p, int idx64, int64_t i) {
    return idx64 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
}

struct PoolQ8 {
    uint8_t* codes; int64_t row_b, head_b;      // strides in bytes (= elements)
    float* scales; int64_t scale_row;           // heads are next to each other
    int64_t rows;
};

// One head row: LPR lanes, 16 elements each (lanes at or beyond D/16 idle).  Loading and storing are apart, so that a lane group has
// several rows' loads in flight.  All lanes of the warp call both.
struct HeadRow { uint4 a, b; };
template <typename T>
__device__ __forceinline__ HeadRow load_head_row(const T* src, int lane_in_row, bool mine) {
    HeadRow h{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if (mine) {
        h.a = ld_nc_v4_keep(src + lane_in_row * 16);
        h.b = ld_nc_v4_keep(src + lane_in_row * 16 + 8);
    }
    return h;
}
template <typename T, int CODE, int LPR>
__device__ __forceinline__ void store_head_row(const HeadRow& h, uint8_t* codes, float* scale, int lane_in_row, bool mine) {
    float x[16];
    uint32_t amax = 0;
    const uint32_t w[8] = {h.a.x, h.a.y, h.a.z, h.a.w, h.b.x, h.b.y, h.b.z, h.b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 f = Cvt<T>::to_f2(w[i]);
        x[2 * i] = f.x; x[2 * i + 1] = f.y;
        amax = max(amax, max(abs_bits(f.x), abs_bits(f.y)));
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (!mine) return;
    const RowScale r = row_scale(amax, CodeTop<CODE>::v);
    uint4 c;
    c.x = pack_codes4<CODE>(x, r.inv, r.finite);
    c.y = pack_codes4<CODE>(x + 4, r.inv, r.finite);
    c.z = pack_codes4<CODE>(x + 8, r.inv, r.finite);
    c.w = pack_codes4<CODE>(x + 12, r.inv, r.finite);
    *reinterpret_cast<uint4*>(codes + lane_in_row * 16) = c;
    if (lane_in_row == 0) *scale = r.scale;
}

constexpr int kQ8Threads = 256;
constexpr int kQ8Rows = 2;             // rows of a lane group in flight

// A pass of a CTA: kQ8Rows times (kQ8Threads / LPR) >> hshift tokens x 1 << hshift heads (hshift: the power of two that covers
// heads2, as far as the CTA's lane groups reach); more heads are further passes over the same tokens.
template <typename T, int CODE, int LPR>
__global__ void __launch_bounds__(kQ8Threads) kv_scatter_q8_kernel(const T* __restrict__ src, int64_t src_row, int64_t src_head,
                                                                   PoolQ8 p, const void* __restrict__ dest, int idx64, int64_t n,
                                                                   int heads2, int hshift, int lanes_used) {
    const int sub = threadIdx.x / LPR, lane_in_row = threadIdx.x % LPR;
    const int tokens = (kQ8Threads / LPR) >> hshift, h0 = sub & ((1 << hshift) - 1);
    for (int64_t base = (int64_t)blockIdx.x * tokens * kQ8Rows; base < n; base += (int64_t)gridDim.x * tokens * kQ8Rows) {
        int64_t t[kQ8Rows], slot[kQ8Rows];
        bool on[kQ8Rows];
#pragma unroll
        for (int u = 0; u < kQ8Rows; ++u) {
            t[u] = base + u * tokens + (sub >> hshift);
            on[u] = t[u] < n;
            slot[u] = on[u] ? idx_at(dest, idx64, t[u]) : 0;
        }
        for (int h = h0; h < heads2 + h0; h += 1 << hshift) {           // the same number of turns for every lane
            HeadRow row[kQ8Rows];
            const bool head_on = h < heads2 && lane_in_row < lanes_used;
#pragma unroll
            for (int u = 0; u < kQ8Rows; ++u)
                row[u] = load_head_row<T>(src + t[u] * src_row + (int64_t)h * src_head, lane_in_row, on[u] && head_on);
            if (h == h0) {
#pragma unroll
                for (int u = 0; u < kQ8Rows; ++u) on[u] = on[u] && q8_slot_ok(slot[u], p.rows, 5, t[u]);
            }
#pragma unroll
            for (int u = 0; u < kQ8Rows; ++u)
                store_head_row<T, CODE, LPR>(row[u], p.codes + slot[u] * p.row_b + (int64_t)h * p.head_b, p.scales + slot[u] * p.scale_row + h,
                                             lane_in_row, on[u] && head_on);
        }
    }
}

// The keep-range form: grid (row chunks, batch); request b keeps rows [range_begin, range_begin + new_len) of its K/V block
// and, when asked, registers their slots.
template <typename T, int CODE, int LPR>
__global__ void __launch_bounds__(kQ8Threads) kv_scatter_register_q8_kernel(
    const int32_t* __restrict__ new_len, const int32_t* __restrict__ range_begin, const int32_t* __restrict__ range_end,
    const int64_t* __restrict__ new_len_cumsum, const T* __restrict__ kv, int64_t kv_row, int64_t kv_head,
    const int32_t* __restrict__ kv_b_start_loc, const int32_t* __restrict__ cur_kv_cache_index, const void* __restrict__ mem_index,
    int idx64, PoolQ8 p, int32_t* __restrict__ req_to_token, int64_t rtt_stride, const int32_t* __restrict__ b_req_idx,
    int64_t num_used, int row_cap, int should_register, int heads2, int hshift, int lanes_used) {
    const int b = blockIdx.y;
    int n_new = new_len[b];
    const int rb = range_begin[b], re = range_end[b];
    if (n_new <= 0 || rb < 0 || re < 0) return;
    if (n_new > row_cap) n_new = row_cap;
    const int64_t base0 = (b > 0 ? new_len_cumsum[b - 1] : 0) + num_used;
    const int64_t src0 = (int64_t)kv_b_start_loc[b] + rb;
    int32_t* rtt = nullptr;
    if (should_register) rtt = req_to_token + (int64_t)b_req_idx[b] * rtt_stride + cur_kv_cache_index[b];
    constexpr int kRowsPerCta = kQ8Threads / LPR;
    const int sub = threadIdx.x / LPR, lane_in_row = threadIdx.x % LPR;
    const int tokens = kRowsPerCta >> hshift, h0 = sub & ((1 << hshift) - 1);
    for (int t0 = blockIdx.x * tokens + (sub >> hshift); ; t0 += gridDim.x * tokens) {
        if (!__syncthreads_or(t0 < n_new)) return;
        const bool on = t0 < n_new;
        const int64_t slot = on ? idx_at(mem_index, idx64, base0 + t0) : 0;
        const T* from = kv + (src0 + (on ? t0 : 0)) * kv_row;
        const bool ok = on && q8_slot_ok(slot, p.rows, 6, base0 + t0);
        for (int hb = 0; hb < heads2; hb += 1 << hshift) {
            const int h = hb + h0;
            const bool mine = ok && h < heads2 && lane_in_row < lanes_used;
            const HeadRow row = load_head_row<T>(from + (int64_t)h * kv_head, lane_in_row, mine);
            store_head_row<T, CODE, LPR>(row, p.codes + slot * p.row_b + (int64_t)h * p.head_b, p.scales + slot * p.scale_row + h,
                                         lane_in_row, mine);
        }
        if (ok && should_register && h0 == 0 && lane_in_row == 0) rtt[t0] = (int32_t)slot;
    }
}

template <typename OT> struct Out16;
template <> struct Out16<__half> {
    static __device__ __forceinline__ void st(__half* o, const float (&x)[16]) {
        uint4 a, b;
        a.x = Cvt<__half>::pack(x[0], x[1]); a.y = Cvt<__half>::pack(x[2], x[3]); a.z = Cvt<__half>::pack(x[4], x[5]); a.w = Cvt<__half>::pack(x[6], x[7]);
        b.x = Cvt<__half>::pack(x[8], x[9]); b.y = Cvt<__half>::pack(x[10], x[11]); b.z = Cvt<__half>::pack(x[12], x[13]); b.w = Cvt<__half>::pack(x[14], x[15]);
        reinterpret_cast<uint4*>(o)[0] = a; reinterpret_cast<uint4*>(o)[1] = b;
    }
};
template <> struct Out16<__nv_bfloat16> {
    static __device__ __forceinline__ void st(__nv_bfloat16* o, const float (&x)[16]) {
        uint4 a, b;
        a.x = Cvt<__nv_bfloat16>::pack(x[0], x[1]); a.y = Cvt<__nv_bfloat16>::pack(x[2], x[3]); a.z = Cvt<__nv_bfloat16>::pack(x[4], x[5]); a.w = Cvt<__nv_bfloat16>::pack(x[6], x[7]);
        b.x = Cvt<__nv_bfloat16>::pack(x[8], x[9]); b.y = Cvt<__nv_bfloat16>::pack(x[10], x[11]); b.z = Cvt<__nv_bfloat16>::pack(x[12], x[13]); b.w = Cvt<__nv_bfloat16>::pack(x[14], x[15]);
        reinterpret_cast<uint4*>(o)[0] = a; reinterpret_cast<uint4*>(o)[1] = b;
    }
};
template <> struct Out16<float> {
    static __device__ __forceinline__ void st(float* o, const float (&x)[16]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(o)[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    }
};

// One lane: 16 codes of a head row.
template <typename OT, int CODE>
__global__ void __launch_bounds__(kQ8Threads) kv_gather_q8_kernel(OT* __restrict__ out, int64_t out_row, int64_t out_head, PoolQ8 p,
                                                                  const void* __restrict__ src, int idx64, int64_t n, int heads2,
                                                                  int vecs) {
    const int per_token = heads2 * vecs;
    const int64_t total = n * per_token;
    for (int64_t i = (int64_t)blockIdx.x * kQ8Threads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kQ8Threads) {
        const int64_t t = i / per_token;
        const int rem = (int)(i - t * per_token);
        const int h = rem / vecs, c = rem - h * vecs;
        const int64_t slot = idx_at(src, idx64, t);
        float x[16];
        if (q8_slot_ok(slot, p.rows, 7, t)) {
            const uint4 w = *reinterpret_cast<const uint4*>(p.codes + slot * p.row_b + (int64_t)h * p.head_b + c * 16);
            const float s = p.scales[slot * p.scale_row + h];
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float f[4];
                unpack_codes4<CODE>(u[j], f);
#pragma unroll
                for (int k = 0; k < 4; ++k) x[4 * j + k] = f[k] * s;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = 0.f;                 // an id outside the pool names no token
        }
        Out16<OT>::st(out + t * out_row + (int64_t)h * out_head + c * 16, x);
    }
}

static int check_pool_q8(const void* codes, int64_t row, int64_t head, const void* scales, int64_t scale_row, int32_t heads2,
                         int32_t head_dim, int32_t code, int64_t pool_rows) {
    if (!codes || !scales || heads2 <= 0 || head_dim <= 0 || pool_rows <= 0) return ESP_ERR_BAD_ARG;
    if (code != ESP_CODE_INT8 && code != ESP_CODE_E4M3) return ESP_ERR_BAD_ARG;
    if (head_dim > 256) return ESP_ERR_UNSUPPORTED;
    if (head_dim % 16 || row % 16 || head % 16 || !aligned16(codes)) return ESP_ERR_ALIGNMENT;
    if (scale_row < heads2 || ((uintptr_t)scales & 3u)) return ESP_ERR_BAD_ARG;
    return ESP_OK;
}

// lanes that share a head row: the power of two that covers head_dim / 16
static int lanes_per_row(int head_dim) {
    int l = 1;
    while (l * 16 < head_dim) l *= 2;
    return l;
}

// log2 of the heads of a pass: the power of two that covers them, within the lane groups of a CTA
static int head_shift(int heads2, int lpr) {
    int h = 0;
    while ((1 << h) < heads2 && (1 << h) < kQ8Threads / lpr) ++h;
    return h;
}

static unsigned q8_grid(int64_t head_rows, int rows_per_cta) {
    const int64_t want = (head_rows + rows_per_cta - 1) / rows_per_cta, cap = (int64_t)kNumSMs * 32;
    return (unsigned)(want < cap ? (want > 0 ? want : 1) : cap);
}

int kv_q8_status(int32_t out[4], int32_t clear) {
    ESP_CUDA_TRY(cudaMemcpyFromSymbol(out, g_kv_q8_status, sizeof(int) * 4));
    if (clear) {
        int zero[4] = {0, 0, 0, 0};
        ESP_CUDA_TRY(cudaMemcpyToSymbol(g_kv_q8_status, zero, sizeof(zero)));
    }
    return ESP_OK;
}

template <typename T, int CODE, int LPR>
static int launch_scatter_q8(const void* src, int64_t sr, int64_t sh, const PoolQ8& p, const void* dest, int idx64, int64_t n, int heads2,
                             int lanes_used, cudaStream_t s) {
    const int hshift = head_shift(heads2, LPR);
    kv_scatter_q8_kernel<T, CODE, LPR><<<q8_grid(n, kQ8Rows * ((kQ8Threads / LPR) >> hshift)), kQ8Threads, 0, s>>>((const T*)src, sr, sh, p, dest, idx64, n, heads2,
                                                                                                      hshift, lanes_used);
    ESP_LAUNCH_CHECK("kv_scatter_q8_kernel");
    return ESP_OK;
}

struct RegisterArgs {
    const int32_t *new_len, *range_begin, *range_end; const int64_t* cumsum; const int32_t *start_loc, *cur; const void* mem_index;
    int idx64; int32_t* rtt; int64_t rtt_stride; const int32_t* b_req_idx; int64_t num_used; int row_cap, should_register; dim3 grid;
};
template <typename T, int CODE, int LPR>
static int launch_register_q8(const RegisterArgs& a, const void* kv, int64_t kr, int64_t kh, const PoolQ8& p, int heads2, int lanes_used, cudaStream_t s) {
    kv_scatter_register_q8_kernel<T, CODE, LPR><<<a.grid, kQ8Threads, 0, s>>>(
        a.new_len, a.range_begin, a.range_end, a.cumsum, (const T*)kv, kr, kh, a.start_loc, a.cur, a.mem_index, a.idx64, p, a.rtt, a.rtt_stride,
        a.b_req_idx, a.num_used, a.row_cap, a.should_register, heads2, head_shift(heads2, LPR), lanes_used);
    ESP_LAUNCH_CHECK("kv_scatter_register_q8_kernel");
    return ESP_OK;
}

}  // namespace esp

using namespace esp;

// CALL(T, CODE, LPR) for the run-time dtype, code type and head width
#define ESP_Q8_LANES(CALL, T, CODE, LPR_)                                                                                        \
    switch (LPR_) {                                                                                                              \
        case 1: return CALL(T, CODE, 1); case 2: return CALL(T, CODE, 2); case 4: return CALL(T, CODE, 4);                        \
        case 8: return CALL(T, CODE, 8); default: return CALL(T, CODE, 16);                    \
    }
#define ESP_Q8_DISPATCH(CALL, dtype, code, LPR_)                                                                                 \
    if (dtype == ESP_DTYPE_F16) {                                                                                                \
        if (code == ESP_CODE_INT8) ESP_Q8_LANES(CALL, __half, ESP_CODE_INT8, LPR_) else ESP_Q8_LANES(CALL, __half, ESP_CODE_E4M3, LPR_) \
    } else {                                                                                                                     \
        if (code == ESP_CODE_INT8) ESP_Q8_LANES(CALL, __nv_bfloat16, ESP_CODE_INT8, LPR_)                                         \
        else ESP_Q8_LANES(CALL, __nv_bfloat16, ESP_CODE_E4M3, LPR_)                                                               \
    }

extern "C" int esp_kv_scatter_q8(const void* src, int64_t src_row_stride, int64_t src_head_stride, void* codes, int64_t codes_row_stride,
                                 int64_t codes_head_stride, float* scales, int64_t scales_row_stride, const void* dest, int32_t idx64,
                                 int64_t n, int32_t heads2, int32_t head_dim, int32_t dtype, int32_t code, int64_t pool_rows, void* stream) {
    if (n == 0) return ESP_OK;
    if (!src || !dest || n < 0) return ESP_ERR_BAD_ARG;
    if (dtype != ESP_DTYPE_F16 && dtype != ESP_DTYPE_BF16) return ESP_ERR_BAD_ARG;
    int rc = check_pool_q8(codes, codes_row_stride, codes_head_stride, scales, scales_row_stride, heads2, head_dim, code, pool_rows);
    if (rc) return rc;
    if (src_row_stride % 8 || src_head_stride % 8 || !aligned16(src)) return ESP_ERR_ALIGNMENT;
    const PoolQ8 p{(uint8_t*)codes, codes_row_stride, codes_head_stride, scales, scales_row_stride, pool_rows};
    cudaStream_t s = (cudaStream_t)stream;
#define ESP_CALL(T, CODE, LPR) launch_scatter_q8<T, CODE, LPR>(src, src_row_stride, src_head_stride, p, dest, idx64, n, heads2, head_dim / 16, s)
    ESP_Q8_DISPATCH(ESP_CALL, dtype, code, lanes_per_row(head_dim))
#undef ESP_CALL
}

extern "C" int esp_kv_scatter_register_q8(
    int32_t batch, const int32_t* new_len, const int32_t* range_begin, const int32_t* range_end, const int64_t* new_len_cumsum,
    const void* kv, int64_t kv_row_stride, int64_t kv_head_stride, const int32_t* kv_b_start_loc, const int32_t* cur_kv_cache_index,
    const void* mem_index, int32_t idx64, void* codes, int64_t codes_row_stride, int64_t codes_head_stride, float* scales,
    int64_t scales_row_stride, int32_t* req_to_token, int64_t req_to_token_stride, const int32_t* b_req_idx, int64_t num_used_mem_index,
    int32_t max_len_in_batch, int32_t should_register, int32_t heads2, int32_t head_dim, int32_t dtype, int32_t code, int64_t pool_rows,
    void* stream) {
    if (batch == 0 || max_len_in_batch <= 0) return ESP_OK;
    if (!new_len || !range_begin || !range_end || !new_len_cumsum || !kv || !kv_b_start_loc || !mem_index || batch < 0) return ESP_ERR_BAD_ARG;
    if (should_register && (!req_to_token || !b_req_idx || !cur_kv_cache_index)) return ESP_ERR_BAD_ARG;
    if (dtype != ESP_DTYPE_F16 && dtype != ESP_DTYPE_BF16) return ESP_ERR_BAD_ARG;
    if (batch > 65535) return ESP_ERR_TOO_LARGE;
    int rc = check_pool_q8(codes, codes_row_stride, codes_head_stride, scales, scales_row_stride, heads2, head_dim, code, pool_rows);
    if (rc) return rc;
    if (kv_row_stride % 8 || kv_head_stride % 8 || !aligned16(kv)) return ESP_ERR_ALIGNMENT;
    const PoolQ8 p{(uint8_t*)codes, codes_row_stride, codes_head_stride, scales, scales_row_stride, pool_rows};
    const int lpr = lanes_per_row(head_dim);
    RegisterArgs a{new_len, range_begin, range_end, new_len_cumsum, kv_b_start_loc, cur_kv_cache_index, mem_index, idx64, req_to_token,
                   req_to_token_stride, b_req_idx, num_used_mem_index, max_len_in_batch > 2147483392 ? 2147483647 : (max_len_in_batch + 255) / 256 * 256, should_register, dim3(1)};
    // the 16-bit form's row cap: rows past max_len_in_batch rounded up to 256 are not copied
    const int64_t per = ((int64_t)kNumSMs * 32 + batch - 1) / batch;
    int64_t gx = q8_grid(max_len_in_batch, (kQ8Threads / lpr) >> head_shift(heads2, lpr));
    a.grid = dim3((unsigned)(gx < per ? gx : per), batch);
    cudaStream_t s = (cudaStream_t)stream;
#define ESP_CALL(T, CODE, LPR) launch_register_q8<T, CODE, LPR>(a, kv, kv_row_stride, kv_head_stride, p, heads2, head_dim / 16, s)
    ESP_Q8_DISPATCH(ESP_CALL, dtype, code, lpr)
#undef ESP_CALL
}

extern "C" int esp_kv_gather_q8(void* out, int64_t out_row_stride, int64_t out_head_stride, const void* codes, int64_t codes_row_stride,
                                int64_t codes_head_stride, const float* scales, int64_t scales_row_stride, const void* src, int32_t idx64,
                                int64_t n, int32_t heads2, int32_t head_dim, int32_t dtype, int32_t code, int64_t pool_rows, void* stream) {
    if (n == 0) return ESP_OK;
    if (!out || !src || n < 0) return ESP_ERR_BAD_ARG;
    int rc = check_pool_q8(codes, codes_row_stride, codes_head_stride, scales, scales_row_stride, heads2, head_dim, code, pool_rows);
    if (rc) return rc;
    const int per16 = dtype == ESP_DTYPE_F32 ? 4 : 8;
    if (out_row_stride % per16 || out_head_stride % per16 || !aligned16(out)) return ESP_ERR_ALIGNMENT;
    const PoolQ8 p{(uint8_t*)const_cast<void*>(codes), codes_row_stride, codes_head_stride, const_cast<float*>(scales), scales_row_stride, pool_rows};
    cudaStream_t s = (cudaStream_t)stream;
    const int vecs = head_dim / 16;
    const unsigned grid = q8_grid(n * heads2 * (int64_t)vecs, kQ8Threads);
#define ESP_G(OT, CODE) kv_gather_q8_kernel<OT, CODE><<<grid, kQ8Threads, 0, s>>>((OT*)out, out_row_stride, out_head_stride, p, src, idx64, n, heads2, vecs)
#define ESP_G2(OT) { if (code == ESP_CODE_INT8) ESP_G(OT, ESP_CODE_INT8); else ESP_G(OT, ESP_CODE_E4M3); }
    if (dtype == ESP_DTYPE_F16) ESP_G2(__half)
    else if (dtype == ESP_DTYPE_BF16) ESP_G2(__nv_bfloat16)
    else if (dtype == ESP_DTYPE_F32) ESP_G2(float)
    else return ESP_ERR_BAD_ARG;
#undef ESP_G2
#undef ESP_G
    ESP_LAUNCH_CHECK("kv_gather_q8_kernel");
    return ESP_OK;
}
