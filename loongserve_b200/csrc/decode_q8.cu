// Split-KV decode attention over a KV pool held in 8 bits (codes and one fp32 scale per slot and head, quant_common.cuh):
//   s_t = (q . ck_t) * k_scale_t * sm_scale,   p_t = exp(s_t - m),   o = sum_t p_t * v_scale_t * cv_t / sum_t p_t
// Stage 1 writes the same splits and partials as the 16-bit form (decode_attention.cu); the call that does both stages divides the
// tokens itself (below).
//
// Bound by HBM: 2 * (128 + 4) bytes per token and kv head, each read once (64 requests x 4096-65536 tokens x 32 kv heads, 17.9 GB:
// 2.74 ms, 6.5 TB/s; the 16-bit pool of the same requests 5.13 ms), and next to that by power: a GPU that runs it without a pause
// lowers its clocks (at 980 W a call of 32 requests x 1K-16K tokens x 32 kv heads takes 15 % longer in a loop than in a burst), so
// instructions per byte count.  At that rate one SM has to take in a code every 1/23 of a cycle and multiply it with up to 8 query heads, which is
// past what fp32 lanes do next to the conversion; the products run on the tensor cores (mma.sync), which are far from their limit
// here.  A lane reads 16-byte pieces of the rows and its pieces ARE operand fragments, because the order of the summed index
// (head dims for S, tokens for O) is free:
//   S [rows 16 x tokens 8] = Q K^T    B fragment of lane (g, c): token g, dims {16c..16c+15, 64+16c..64+16c+15}; Q fragments are
//                                     loaded once in the same dim order.
//   O^T [dims 16 x heads 8] += V^T P^T  A fragment of lane (g, c): dims 16g..16g+15, tokens 2c, 2c+1, 2c+8, 2c+9 (words of two
//                                     tokens interleaved byte by byte); P^T's fragment is what the lane holds of S.
// (lane = 4g + c.)  A warp takes 16 tokens of one head tile per step.
//
// Precision.  Scores, maxima, sums and outputs are fp32.
//   S, int8 codes: they are operands as they lie in the pool (m16n8k32, 32-bit integer sums); q, scaled by a power of two per head, is
//   an integer of 30 bits in four balanced base-256 digits, rows j, j + 4, j + 8, j + 12 of A (groups of up to four heads, GT = 4), or
//   of 22 bits in three (GT = 8: rows j, j + 8, and a second product).  Against codes brought to f16 this saves a third of the
//   instructions: 477 us instead of 499 for the 32 requests above, in a loop, before the copies were what they are now.
//   S, e4m3 codes: brought to f16 (exactly; two instructions a word), q scaled to 2^7 in f16, exact down to 2^-21 of its largest.
//   O: codes become f16 (exactly: 8 bits fit).  A weight p * v_scale enters in units of 2^-12 * v_ref, v_ref 1 to 4 times the largest v_scale
//   that the warp has seen, as its rounding to f16 and the rounding of what that left: 2^-22 relative, and at least 2^-37 of v_ref (below f16's
//   normal range), so that a token whose v_scale is far below the largest has fewer bits.  (The rounding alone, 2^-12, showed in f16 outputs: 3.3e-4
//   against 2.0e-4 for fp32 weights.)  With GT = 4 the rests take the columns of heads 4-7 and cost no product; GT = 8 multiplies V
//   twice.
#include <algorithm>
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
    float scale_log2; int64_t pool_rows;
    int max_len, num_blocks, counted, ranges, min_units;  // ranges > 0: the tokens of all requests in that many equal pieces
    int* parts;                                  // ranges: per request its first piece's partial and how many it has
    int head_tiles, head_groups, scale_vec, q_bf16;      // tiles of up to 8 q heads of one kv head; CTAs that cover them all for one split
    void* o; float* lse; int o_dtype, direct;    // results; direct: one split per request, whose results are written at once
};

constexpr int kQ8Warps = 4, kQ8HeadTile = 8;
constexpr int kQ8Resident = 3 * kNumSMs, kQ8MinPiece = 64;       // CTAs the GPU holds; tokens below which a piece is not cut
// requests up to this length are not cut at all (measured at the call that uses it)
inline int q8_whole(int batch) { return batch < 8 ? 256 : 512; }

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// A CTA covers NH neighbouring kv heads (or one group of 8 q heads of one kv head) and one split of the tokens: its four consumer
// warps are NH heads x WT = 4 / NH interleaved shares of the split's tokens.  A fifth warp fetches, with 16-byte asynchronous
// copies: one instruction takes the NH heads' K (or V) codes of WT tokens, 512 contiguous bytes for NH = 4, into a ring of
// stages of 16 * WT tokens, counted on mbarriers.  Against fetches by the consumer warps themselves this takes address
// arithmetic and slot lookups out of their instruction streams, and a scale's 32-byte sector is asked for once per CTA instead
// of once per head.  (One bulk copy per token and operand instead: 81 cycles each from one warp, 3.3 TB/s at best.)  A row lies
// in shared memory as in the pool, a 128-byte line to a line, with its eight 16-byte pieces in another order (k_piece, v_piece),
// so that the fragment reads (16 bytes per lane) have no bank conflicts.  Rows at odd pitches would do for the banks too, but a
// copy whose line ends up across two lines of shared memory asks the L2 for the sectors on the border twice: half as many again.
//
// CTAs are persistent: each walks over items (a request's tokens t0..t1, heads), and the producer runs ahead into the next item, so
// that neither the start of an item (length, slots, queries) nor its results stop the flow of copies.  How the tokens are divided:
//   ranges   the steps of all requests, laid end to end, are cut into as many equal pieces as there are CTAs for each group of heads;
//            a piece that crosses requests has an item for each.  Pieces and requests both only grow along the way, so piece + request
//            numbers a partial uniquely, and there are at most pieces + requests of them.  A request inside one piece gets its results
//            at once.  Against splits of a fixed length every CTA has the same work and writes a partial or two instead of one per
//            128 to 512 tokens: 185 us instead of 195 (the best length) to 241 for 2 requests x 8 kv heads (group 4), 501702 tokens; 66
//            instead of 76 to 80 for 64 requests x 4096 tokens x 4 kv heads (group 8); 392 instead of 389 (splits of 512) to 467 (of 128)
//            for 32 requests x 32 kv heads, 287567 tokens.
//   counted  splits of seq_block_size tokens, where a CTA has several and the batch is small enough: those that exist are counted
//            first, so that ragged batches divide evenly.
//   else     all splits up to the longest possible request; those behind a request's end are passed over.
constexpr int kQ8MaxCounted = 384;        // requests whose lengths are held in shared memory
struct WarpStateQ8 { float acc[32][32], m[32], l[32], v[32]; };      // [register][lane]
template <int NH> struct RingQ8 {
    static constexpr int WT = kQ8Warps / NH, kTokens = 16 * WT;
    static constexpr int kPitch = NH * 128, kOffV = kTokens * kPitch;
    static constexpr int kOffScale = 2 * kOffV;                                                 // scales [K, V][token][NH]
    static constexpr int kOffPresent = kOffScale + 2 * kTokens * NH * 4;                        // WT masks of 16 tokens
    static constexpr int kStageBytes = kOffPresent + 128;
    static constexpr int kStages = NH == 4 ? 4 : 3;
    static constexpr int kOffBar = kStages * kStageBytes;                                       // full [kStages], empty [kStages]
    static constexpr int kOffAbort = kOffBar + 2 * kStages * 8;
    static constexpr int kOffMerge = kOffAbort + 16;                                            // states of the warps with wt > 0
    static constexpr int kOffLen = kOffMerge + (WT - 1) * NH * (int)sizeof(WarpStateQ8);        // lengths, first blocks
    static constexpr int kSmem = kOffLen + (2 * kQ8MaxCounted + 1) * 4;
};
static_assert(3 * (RingQ8<4>::kSmem + 1024) <= 233472 && 3 * (RingQ8<2>::kSmem + 1024) <= 233472 && 3 * (RingQ8<1>::kSmem + 1024) <= 233472,
              "three CTAs to an SM");

// copies 16 or 4 bytes, or fills them with zeros
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool have) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(have ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool have) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(have ? 4 : 0) : "memory");
}
// one arrival (of the barrier's count) once this thread's asynchronous copies so far have landed
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// Limit of the mbarrier waits in SM cycles; on expiry {ESP_ERR_DEVICE_TIMEOUT, block, which (8 producer, 9 consumer), step} is
// recorded, the CTA writes no results, and later launches return at once until the status has been read.
__device__ long long g_decode_q8_wait_limit_cycles = 2000000000LL;
__device__ __noinline__ void q8_timeout(int which, int step) {
    int old = atomicCAS(&g_decode_q8_status[0], 0, ESP_ERR_DEVICE_TIMEOUT);
    if (old == ESP_ERR_BAD_SLOT) old = atomicCAS(&g_decode_q8_status[0], ESP_ERR_BAD_SLOT, ESP_ERR_DEVICE_TIMEOUT) == ESP_ERR_BAD_SLOT ? 0 : 1;
    if (old == 0) {                                  // results that are missing come before a token that was left out
        g_decode_q8_status[1] = blockIdx.x + gridDim.x * blockIdx.y;
        g_decode_q8_status[2] = which;
        g_decode_q8_status[3] = step;
    }
}
__device__ __forceinline__ bool q8_wait(uint32_t bar, uint32_t parity, volatile int* abort, int which, int step) {
    const int r = ptx::mbar_wait_bounded(bar, parity, &g_decode_q8_wait_limit_cycles, abort);
    if (r == 2) { q8_timeout(which, step); *abort = 1; }
    return r == 0;
}

__device__ __forceinline__ void store_as(void* o, int64_t i, float x, int dtype) {
    if (dtype == ESP_DTYPE_F32) reinterpret_cast<float*>(o)[i] = x;
    else if (dtype == ESP_DTYPE_F16) reinterpret_cast<__half*>(o)[i] = __float2half_rn(x);
    else reinterpret_cast<__nv_bfloat16*>(o)[i] = __float2bfloat16_rn(x);
}

// 16 values of an output row
__device__ __forceinline__ void store_row16(void* o, int64_t i, const float (&x)[16], int dtype) {
    if (dtype == ESP_DTYPE_F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) reinterpret_cast<float4*>(reinterpret_cast<float*>(o) + i)[j] = make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
        return;
    }
    uint32_t u[8];
    if (dtype == ESP_DTYPE_F16) {
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = Cvt<__half>::pack(x[2 * j], x[2 * j + 1]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = Cvt<__nv_bfloat16>::pack(x[2 * j], x[2 * j + 1]);
    }
    uint4* p = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(o) + i);
    p[0] = make_uint4(u[0], u[1], u[2], u[3]); p[1] = make_uint4(u[4], u[5], u[6], u[7]);
}

// where piece i of 16 bytes of a head's row lies, by the row's token
__device__ __forceinline__ int k_piece(int i, int token) { return i ^ (token & 1) << 2; }
__device__ __forceinline__ int v_piece(int i, int token) { return i ^ (token & 6); }

struct ItemQ8 { int b, hg, t0, t1, req, steps; int64_t row0; bool write, whole; };   // row0: of the partials, in rows of all heads
struct CursorQ8 { int n, u, u1; };             // (piece, heads), its units from u to u1 are still to do

template <int CODE, int NH, int GT>
__global__ void __launch_bounds__(kQ8Warps * 32 + 32, 3) decode_stage1_q8_kernel(DecodeQ8Args a) {
    using R = RingQ8<NH>;
    constexpr int WT = R::WT;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t sbase = ptx::smem_u32(smem);
    auto full = [sbase](int st) { return sbase + R::kOffBar + 8u * st; };
    auto empty = [sbase](int st) { return sbase + R::kOffBar + 8u * (R::kStages + st); };
    volatile int* s_abort = reinterpret_cast<volatile int*>(smem + R::kOffAbort);
    int* s_len = reinterpret_cast<int*>(smem + R::kOffLen);               // -1: the request's row is not in the table
    int* s_first = s_len + kQ8MaxCounted;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == kQ8Warps * 32) {                                   // not a thread that waits for the first lengths
        s_abort[0] = s_abort[1] = *reinterpret_cast<volatile int*>(&g_decode_q8_status[0]) == ESP_ERR_DEVICE_TIMEOUT ? 1 : 0;
        for (int i = 0; i < R::kStages; ++i) { ptx::mbar_init(full(i), 33); ptx::mbar_init(empty(i), kQ8Warps); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // The queries, the pool and the lengths are there from here on; what is above may run while the kernel ahead ends (one request of
    // 512 tokens 10.1 -> 9.3 us, 64 of up to 512 18.1 -> 17.5).  Neither this kernel nor the merge lets the next one start earlier than
    // that: CTAs placed while some SMs are still busy end up uneven (that 19.5 us; two requests in splits of 4096 tokens 237 -> 320).
    grid_dependency_wait();
    auto blocks_of = [&](int len) { return len <= 0 ? 0 : min((len - 1) / a.seq_block_size + 1, a.num_blocks); };
    const int unit = a.ranges ? R::kTokens : a.seq_block_size;
    if (a.counted) {
        for (int b = threadIdx.x; b < a.batch; b += blockDim.x) {
            const int len = a.b_seqlen[b], req = a.b_req_idx[b];
            const bool ok = req >= 0 && req < a.rtt_rows && len <= a.rtt_cols;
            if (!ok && len > 0) q8_report(1, req);
            const int seen = min(len, a.max_len);
            s_len[b] = ok ? (a.ranges ? seen : len) : -1;
            s_first[b + 1] = a.ranges ? (seen <= 0 ? 0 : (seen - 1) / R::kTokens + 1) : blocks_of(len);
        }
        __syncthreads();
        if (warp == 0) {
            int carry = 0;
            for (int b0 = 0; b0 < a.batch; b0 += 32) {
                int x = b0 + lane < a.batch ? s_first[b0 + lane + 1] : 0;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
                if (b0 + lane < a.batch) s_first[b0 + lane + 1] = carry + x;
                carry += __shfl_sync(0xffffffffu, x, 31);
            }
            if (lane == 0) s_first[0] = 0;
        }
    }
    __syncthreads();
    const int units = a.counted ? s_first[a.batch] : a.num_blocks * a.batch;
    const int per = a.ranges ? max(a.min_units, (units - 1) / a.ranges + 1) : 1;
    const int items = (units == 0 ? 0 : (units - 1) / per + 1) * a.head_groups;
    if (a.ranges && blockIdx.x == 0)
        for (int b = threadIdx.x; b < a.batch; b += blockDim.x) {
            const int u0 = s_first[b], u1 = s_first[b + 1];
            a.parts[2 * b] = u0 / per + b;
            a.parts[2 * b + 1] = u1 > u0 ? (u1 - 1) / per - u0 / per + 1 : 0;
        }
    // The next item of a cursor.  All head groups of a piece are neighbouring CTAs' work: their rows are neighbours in memory.
    CursorQ8 cur{(int)blockIdx.x - (int)gridDim.x, 0, 0};
    auto next_item = [&](ItemQ8& it) -> bool {
        if (cur.u >= cur.u1) {
            cur.n += gridDim.x;
            if (cur.n >= items) return false;
            cur.u = cur.n / a.head_groups * per;
            cur.u1 = min(cur.u + per, units);
        }
        const int piece = cur.n / a.head_groups;
        it.hg = cur.n - piece * a.head_groups;
        int len;
        if (a.counted) {
            int lo = 0, hi = a.batch - 1;                                 // the last request whose first unit is not behind u
            while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (s_first[mid] <= cur.u) lo = mid; else hi = mid - 1; }
            const int first = s_first[lo], behind = s_first[lo + 1], end = min(cur.u1, behind);
            it.b = lo;
            len = s_len[lo];
            it.req = len > 0 ? a.b_req_idx[lo] : 0;
            it.write = true;
            it.whole = a.ranges && cur.u == first && end == behind;
            it.t0 = (cur.u - first) * unit;
            it.t1 = min((end - first) * unit, len);
            it.row0 = it.whole ? lo : (a.ranges ? piece + lo : (int64_t)(cur.u - first) * a.batch + lo);
            cur.u = end;
        } else {
            it.b = cur.u / a.num_blocks;
            const int blk = cur.u - it.b * a.num_blocks;
            len = a.b_seqlen[it.b];
            it.req = a.b_req_idx[it.b];
            it.write = a.direct || blk < blocks_of(len);
            it.whole = a.direct;
            if (len > 0 && (it.req < 0 || it.req >= a.rtt_rows || len > a.rtt_cols)) {
                if (threadIdx.x == 0) q8_report(1, it.req);
                len = 0;
            }
            it.t0 = blk * unit;
            it.t1 = min(it.t0 + unit, len);
            it.row0 = (int64_t)blk * a.batch + it.b;
            ++cur.u;
        }
        it.steps = it.t1 > it.t0 ? (it.t1 - it.t0 + R::kTokens - 1) / R::kTokens : 0;
        return true;
    };
    const int tiles_per_kv = (a.group + kQ8HeadTile - 1) / kQ8HeadTile;   // more than 1 only with NH = 1

    if (warp == kQ8Warps) {
        // ------------------------------------------------------------------ producer
        const int tok = lane & 15, isv = lane >> 4;
        const int piece = lane % (NH * 8), share = lane / (NH * 8);         // 16 bytes of a row; which of an instruction's WT tokens
        const int64_t ssrc_stride = isv ? a.vs_stride_t : a.ks_stride_t;
        bool ok = !s_abort[1];
        int done = 0, st = 0, phase = 1;                                  // the first pass over the ring finds it empty
        ItemQ8 it;
        while (ok && next_item(it)) {
          const int kv0 = it.hg * NH / tiles_per_kv;
          const int32_t* rtt = a.req_to_tokens + (it.steps > 0 ? (int64_t)it.req * a.rtt_stride : 0);
          const uint8_t* ksrc = a.k + (int64_t)kv0 * a.k_stride_h + piece * 16;
          const uint8_t* vsrc = a.v + (int64_t)kv0 * a.v_stride_h + piece * 16;
          const float* ssrc = isv ? a.v_scale + kv0 : a.k_scale + kv0;
          // Slots of steps i (lanes 0-15) and i + 1 (lanes 16-31), 16 tokens of share u.  They are asked for eight steps at a time (four
          // with NH < 4), as many steps before they are looked at: they queue behind the copies, and looking at one waits for all that
          // have been asked for.  (Looked at when asked for: two thirds of the producer's time; two steps at a time: half of it.)
          auto token_of = [&](int i, int u) { return it.t0 + ((i + isv) * WT + u) * 16 + tok; };
          auto ask = [&](int i, int u) -> int {
            const int t = token_of(i, u);
            return i + isv < it.steps && t < it.t1 ? rtt[t] : 0;
          };
          auto check = [&](int i, int u, int s) -> int {                  // -1: no such token
            if (i + isv >= it.steps || token_of(i, u) >= it.t1) return -1;
            if (s < 0 || s >= a.pool_rows) { q8_report(0, s); return -1; }
            return s;
          };
          constexpr int kPairs = NH == 4 ? 4 : 2;
          int slots[kPairs][WT], later[kPairs][WT];
#pragma unroll
          for (int k = 0; k < kPairs; ++k)
#pragma unroll
              for (int u = 0; u < WT; ++u) later[k][u] = ask(2 * k, u);
          for (int i = 0; i < it.steps; ++i, ++done) {
            ok = __all_sync(0xffffffffu, q8_wait(empty(st), phase, s_abort, 8, done));
            if (!ok) break;
            const uint32_t stage = sbase + st * R::kStageBytes;
            if (i % (2 * kPairs) == 0) {
#pragma unroll
                for (int k = 0; k < kPairs; ++k)
#pragma unroll
                    for (int u = 0; u < WT; ++u) slots[k][u] = check(i + 2 * k, u, later[k][u]);
            }
            const int pair = i / 2 % kPairs;
            int s[WT];
#pragma unroll
            for (int u = 0; u < WT; ++u) {
                int mine = slots[0][u];
#pragma unroll
                for (int k = 1; k < kPairs; ++k) mine = pair == k ? slots[k][u] : mine;
                s[u] = __shfl_sync(0xffffffffu, mine, (i & 1) * 16 + tok);
                const uint32_t present = __ballot_sync(0xffffffffu, s[u] >= 0) & 0xffffu;
                if (lane == 0) *reinterpret_cast<uint32_t*>(smem + st * R::kStageBytes + R::kOffPresent + 4 * u) = present;
            }
            if (lane == 0) ptx::mbar_arrive(full(st));                // publishes the masks
#pragma unroll
            for (int j = 0; j < 16; ++j) {                            // tokens j * WT + share; absent ones are filled with zeros
                const int slot = __shfl_sync(0xffffffffu, s[j * WT / 16], j * WT % 16 + share);
                const int64_t row = max(slot, 0);
                const uint32_t at = j * WT + share;
                const uint32_t line = stage + at * R::kPitch + (piece >> 3) * 128;
                cp_async16(line + k_piece(piece & 7, at) * 16, ksrc + row * a.k_stride_t, slot >= 0);
                cp_async16(line + R::kOffV + v_piece(piece & 7, at) * 16, vsrc + row * a.v_stride_t, slot >= 0);
            }
#pragma unroll
            for (int u = 0; u < WT; ++u) {                            // scales: lanes 0-15 K, lanes 16-31 V of 16 tokens
                const uint32_t sd = stage + R::kOffScale + ((isv * R::kTokens + u * 16 + tok) * NH) * 4;
                const float* sp = ssrc + (int64_t)max(s[u], 0) * ssrc_stride;
                if (NH == 4 && a.scale_vec) cp_async16(sd, sp, s[u] >= 0);
                else
#pragma unroll
                    for (int h = 0; h < NH; ++h) cp_async4(sd + 4 * h, sp + h, s[u] >= 0);
            }
            cp_async_arrive(full(st));
            if (i % (2 * kPairs) == 0) {
#pragma unroll
                for (int k = 0; k < kPairs; ++k)
#pragma unroll
                    for (int u = 0; u < WT; ++u) later[k][u] = ask(i + 2 * kPairs + 2 * k, u);
            }
            if (++st == R::kStages) { st = 0; phase ^= 1; }
          }
        }
        // whichever warp gives up, the CTA does not leave before the copies have landed (bounded)
        for (int j = done > R::kStages ? done - R::kStages : 0; j < done; ++j)
            ptx::mbar_wait_bounded(full(j % R::kStages), (j / R::kStages) & 1, &kDrainLimitCycles, nullptr);
        return;
    }
    const int g = lane >> 2, c = lane & 3;
    const int hw = warp % NH, wt = warp / NH;            // kv head within the CTA, share of its tokens
    // s_abort[1] keeps its first value: the four warps meet at barriers inside the loop, so all of them enter it or none does, also where
    // one has given up before another has come this far
    bool ok = !s_abort[1];
    int st = 0, phase = 0, done = 0;

    ItemQ8 it;
    while (ok && next_item(it)) {
    if (!it.write) continue;                             // a split behind the request's end: no steps either
    // head tiles of this CTA: kv heads kv0 .. kv0 + NH - 1, or (a group of more than 8 q heads, NH = 1) tile `sub` of one
    const int kv0 = it.hg * NH / tiles_per_kv, sub = it.hg * NH - kv0 * tiles_per_kv;
    const int nheads = min(kQ8HeadTile, a.group - sub * kQ8HeadTile);
    const int h0 = (kv0 + hw) * a.group + sub * kQ8HeadTile;

    // Q fragments, dims in the order of the K words
    constexpr bool kInt = CODE == ESP_CODE_INT8;
    constexpr int kQExp = !kInt ? 7 : (GT == 4 ? 29 : 21);
    uint32_t qf[8][kInt ? (GT == 4 ? 2 : 3) : 2];
    float qs;
    {
        float x[32];
        uint32_t amax = 0;
        const int j = g % GT;
        const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + ((int64_t)it.b * a.num_q_heads + h0 + j) * 128 + c * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 u = j < nheads ? *reinterpret_cast<const uint4*>(qp + (i >> 1) * 64 + (i & 1) * 8) : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 f = a.q_bf16 ? Cvt<__nv_bfloat16>::to_f2(w[k]) : Cvt<__half>::to_f2(w[k]);
                x[8 * i + 2 * k] = f.x; x[8 * i + 2 * k + 1] = f.y;
                amax = max(amax, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
            }
        }
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const bool finite = amax < 0x7f800000u;              // a query with inf or NaN: NaN
        // 2^(kQExp - e) with 2^e <= max|q| < 2^(e + 1): the scaled query lies below 2^(kQExp + 1), which the digits below hold.  e is at
        // least -90, so that both powers are normal numbers, and at most 127 (the largest exponent of bf16), where they are normal too.
        const int e = max((int)(min(amax, 0x7f7fffffu) >> 23) - 127, -90);
        const float up = __uint_as_float((uint32_t)(127 + kQExp - e) << 23);
        qs = finite ? a.scale_log2 * __uint_as_float((uint32_t)(127 - kQExp + e) << 23) : __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if constexpr (kInt) {
                // balanced digits, -128 to 127 each: with 128 added to every lower digit the bytes are digit + 128
                uint32_t v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = ((uint32_t)__float2int_rn(finite ? x[4 * k + i] * up : 0.f) + 0x00808080u) ^ 0x00808080u;
                if constexpr (GT == 4) {                     // lanes of rows 0-3: digits 0 and 2; of rows 4-7: 1 and 3
                    const uint32_t sel = g < 4 ? 0x6240 : 0x7351;
                    const uint32_t t0 = __byte_perm(v[0], v[1], sel), t1 = __byte_perm(v[2], v[3], sel);
                    qf[k][0] = __byte_perm(t0, t1, 0x5410); qf[k][1] = __byte_perm(t0, t1, 0x7632);
                } else {
                    const uint32_t t0 = __byte_perm(v[0], v[1], 0x5140), t1 = __byte_perm(v[2], v[3], 0x5140);
                    qf[k][0] = __byte_perm(t0, t1, 0x5410); qf[k][1] = __byte_perm(t0, t1, 0x7632);
                    qf[k][2] = __byte_perm(__byte_perm(v[0], v[1], 0x0062), __byte_perm(v[2], v[3], 0x0062), 0x5410);
                }
            } else {
                qf[k][0] = Cvt<__half>::pack(x[4 * k] * up, x[4 * k + 1] * up);
                qf[k][1] = Cvt<__half>::pack(x[4 * k + 2] * up, x[4 * k + 3] * up);
            }
        }
    }

    float acc[8][4] = {};                 // MMA j: dims 16g + 2j (0, 1) and 16g + 2j + 1 (2, 3) of heads 2c, 2c + 1
    float m_ref = -INFINITY, l_run = 0.f; // of head g; l over this lane's tokens only
    float v_ref = 0.f, v_mul = 0.f;       // weights are held as p * v_scale * v_mul, v_mul = 2^12 / v_ref, v_ref >= every v_scale so far

    auto compute = [&](const uint8_t* d) {
        const uint8_t* krow = d + (wt * 16 + g) * R::kPitch + hw * 128 + k_piece(c, g) * 16;
        const uint8_t* vrow = d + R::kOffV + (wt * 16 + 2 * c) * R::kPitch + hw * 128 + v_piece(g, 2 * c) * 16;
        const float* scl = reinterpret_cast<const float*>(d + R::kOffScale) + wt * 16 * NH + hw;
        const uint32_t present = *reinterpret_cast<const uint32_t*>(d + R::kOffPresent + 4 * wt);
        float sc[4], vs[4];               // of tokens 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 x = *reinterpret_cast<const uint4*>(krow + 8 * i * R::kPitch);
            const uint4 y = *reinterpret_cast<const uint4*>(krow + 8 * i * R::kPitch + (g & 1 ? -64 : 64));
            const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
            if constexpr (kInt) {
                // a sum of 128 products of a digit and a code is below 2^21: counted in the last places of 1.5 * 2^23, it is a float
                constexpr int kBase = 0x4b400000;
                constexpr float kZero = 12582912.f;
                int d[4] = {kBase, kBase, kBase, kBase}, d2[4] = {kBase, kBase, 0, 0};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    mma_s8(d, qf[2 * j][0], qf[2 * j][1], qf[2 * j + 1][0], qf[2 * j + 1][1], w[2 * j], w[2 * j + 1]);
                    if constexpr (GT == 8) mma_s8(d2, qf[2 * j][2], 0u, qf[2 * j + 1][2], 0u, w[2 * j], w[2 * j + 1]);
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float lo = __int_as_float(d[k]) - kZero, hi = __int_as_float(d[2 + k]) - kZero;
                    if constexpr (GT == 4) {                  // digits 0 and 2 here, 1 and 3 in the lane of row g ^ 4
                        float u = fmaf(hi, 65536.f, lo);
                        u = g < 4 ? u : 256.f * u;
                        sc[2 * i + k] = u + __shfl_xor_sync(0xffffffffu, u, 16);
                    } else {
                        sc[2 * i + k] = fmaf(__int_as_float(d2[k]) - kZero, 65536.f, fmaf(hi, 256.f, lo));
                    }
                }
            } else {
                float s[4] = {};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    uint32_t lo, hi;
                    codes_to_f16<CODE>(w[j], lo, hi);
                    mma_f16(s, qf[j][0], 0u, qf[j][1], 0u, lo, hi);
                }
                sc[2 * i] = s[0]; sc[2 * i + 1] = s[1];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = 2 * c + (i & 1) + 8 * (i >> 1);
            sc[i] *= scl[t * NH] * qs;
            vs[i] = scl[(R::kTokens + t) * NH];
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
        // a weight is its f16 rounding plus the f16 rounding of what that left
        uint32_t b0 = Cvt<__half>::pack(wgt[0], wgt[1]), b1 = Cvt<__half>::pack(wgt[2], wgt[3]);
        const float2 r0 = Cvt<__half>::to_f2(b0), r1 = Cvt<__half>::to_f2(b1);
        const uint32_t e0 = Cvt<__half>::pack(wgt[0] - r0.x, wgt[1] - r0.y), e1 = Cvt<__half>::pack(wgt[2] - r1.x, wgt[3] - r1.y);
        if (GT == 4 && g >= 4) { b0 = e0; b1 = e1; }
        uint32_t vw[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) { const uint4 x = *reinterpret_cast<const uint4*>(vrow + ((i & 1) + 8 * (i >> 1)) * R::kPitch); vw[i][0] = x.x; vw[i][1] = x.y; vw[i][2] = x.z; vw[i][3] = x.w; }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {                      // dims 4w + 2h, 4w + 2h + 1 of this lane's 16
                const uint32_t sel = h ? 0x7362 : 0x5140;
                uint32_t x0, x1, y0, y1;
                codes_to_f16<CODE>(__byte_perm(vw[0][w], vw[1][w], sel), x0, x1);
                codes_to_f16<CODE>(__byte_perm(vw[2][w], vw[3][w], sel), y0, y1);
                mma_f16(acc[2 * w + h], x0, x1, y0, y1, b0, b1);
                if constexpr (GT == 8) mma_f16(acc[2 * w + h], x0, x1, y0, y1, e0, e1);
            }
        }
    };

#pragma unroll 1
    for (int i = 0; i < it.steps; ++i, ++done) {
        ok = __all_sync(0xffffffffu, q8_wait(full(st), phase, s_abort, 9, done));
        if (!ok) break;
        compute(smem + st * R::kStageBytes);
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(empty(st));
        if (++st == R::kStages) { st = 0; phase ^= 1; }
    }
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
    if constexpr (WT > 1) {
        // the shares of a head's tokens meet in the warp with wt = 0; every state is in units of its own references
        WarpStateQ8* ms = reinterpret_cast<WarpStateQ8*>(smem + R::kOffMerge);
        if (wt > 0) {
            WarpStateQ8& w = ms[(wt - 1) * NH + hw];
#pragma unroll
            for (int j = 0; j < 32; ++j) w.acc[j][lane] = acc[j >> 2][j & 3];
            w.m[lane] = m_ref; w.l[lane] = l_run; w.v[lane] = v_ref;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");                    // the four consumer warps
        if (wt == 0) {
#pragma unroll 1
            for (int k = 0; k < WT - 1; ++k) {
                const WarpStateQ8& w = ms[k * NH + hw];
                const float m_new = fmaxf(m_ref, w.m[lane]), m_use = m_new == -INFINITY ? 0.f : m_new;
                const float f0 = exp2f(m_ref - m_use), f1 = exp2f(w.m[lane] - m_use);     // 0 for a warp that saw no token
                const float v_new = fmaxf(v_ref, w.v[lane]);
                // with no value scale above zero on either side both accumulators are zero
                const float r0 = v_new > 0.f ? f0 * (v_ref / v_new) : f0, r1 = v_new > 0.f ? f1 * (w.v[lane] / v_new) : f1;
                l_run = l_run * f0 + w.l[lane] * f1;
                m_ref = m_new; v_ref = v_new;
                const float x0 = __shfl_sync(0xffffffffu, r0, 8 * c), x1 = __shfl_sync(0xffffffffu, r0, 8 * c + 4);
                const float y0 = __shfl_sync(0xffffffffu, r1, 8 * c), y1 = __shfl_sync(0xffffffffu, r1, 8 * c + 4);
#pragma unroll
                for (int j = 0; j < 32; ++j) acc[j >> 2][j & 3] = acc[j >> 2][j & 3] * (j & 1 ? x1 : x0) + w.acc[j][lane] * (j & 1 ? y1 : y0);
            }
        }
        // the states may be written again; the four warps go on, or leave, together
        int leave;
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbar.red.or.pred q, 1, 128, p;\n\tselp.s32 %0, 1, 0, q;\n\t}"
                     : "=r"(leave) : "r"(ok ? 0 : 1) : "memory");
        ok = leave == 0;
    }
    if (ok && wt == 0) {
        const float f = l_run == 0.f ? 0.f : (v_ref * (1.f / 4096.f)) / l_run;            // of head g; no token: zeros
        const float lse = l_run == 0.f ? -INFINITY : ((m_ref == -INFINITY ? 0.f : m_ref) + log2f(l_run)) * kLn2Q8;
        const int64_t row0 = it.row0 * a.num_q_heads + h0;
        if constexpr (GT == 4) {                                          // roundings and rests meet
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[j >> 2][j & 3] += __shfl_xor_sync(0xffffffffu, acc[j >> 2][j & 3], 2);
        }
        if (c == 0 && g < nheads) (it.whole ? a.lse : a.mid_lse)[row0 + g] = lse;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float fk = __shfl_sync(0xffffffffu, f, 8 * c + 4 * k);
            if (2 * c + k < nheads) {
                float x[16];
#pragma unroll
                for (int j = 0; j < 8; ++j) { x[2 * j] = acc[j][k] * fk; x[2 * j + 1] = acc[j][2 + k] * fk; }
                store_row16(it.whole ? a.o : a.mid_o, (row0 + 2 * c + k) * 128 + 16 * g, x, it.whole ? a.o_dtype : ESP_DTYPE_F32);
            }
        }
    }
    }
}

// The partials of one (request, head), by a CTA: at few rows and many splits (two requests of 262144 tokens: 64 rows x 410 splits)
// one warp per row leaves most of the GPU idle (130 us; four warps 31 us).  Warp w takes splits w, w + W, ...; lanes hold four
// dims each.
template <int W>
__global__ void __launch_bounds__(W * 32) decode_merge_q8_kernel(void* o, float* lse, const int32_t* b_seqlen,
                                                                 const float* mid_o, const float* mid_lse, const int* parts,
                                                                 int batch, int num_heads, int num_blocks, int block_seq, int o_dtype) {
    const int pair = blockIdx.x, b = pair / num_heads, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dependency_wait();                                    // its loads pass the L1: it may have started before stage 1 ended
    int n;
    int64_t bh, row0;                                          // rows from one split to the next, row of the first
    if (parts != nullptr) {
        n = __ldcg(parts + 2 * b + 1);
        if (n == 1) return;                                    // stage 1 has written the results
        bh = num_heads;
        row0 = (int64_t)__ldcg(parts + 2 * b) * num_heads + (pair - b * num_heads);
    } else {
        const int len = __ldcg(b_seqlen + b);
        n = len <= 0 ? 0 : min((len - 1) / block_seq + 1, num_blocks);
        bh = (int64_t)batch * num_heads;
        row0 = pair;
    }
    __shared__ float s_m[W], s_l[W], s_o[W][128];
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j0 = warp; j0 < n; j0 += W * 32) {                // up to 32 splits of this warp at a time, one lse per lane
        const int j = j0 + W * lane;
        const float x = j < n ? __ldcg(mid_lse + j * bh + row0) : -INFINITY;
        float mx = x;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        const float m_new = fmaxf(m, mx), m_use = m_new == -INFINITY ? 0.f : m_new;
        const float al = exp2f((m - m_use) * kLog2eQ8), w = exp2f((x - m_use) * kLog2eQ8);
        l = l * al + w;                                        // this lane's share of the sum
        acc.x *= al; acc.y *= al; acc.z *= al; acc.w *= al;
        m = m_new;
        const int cnt = min(32, (n - j0 + W - 1) / W);
#pragma unroll 8
        for (int i = 0; i < cnt; ++i) {
            const float wi = __shfl_sync(0xffffffffu, w, i);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(mid_o + ((int64_t)(j0 + W * i) * bh + row0) * 128 + lane * 4));
            acc.x = fmaf(wi, v.x, acc.x); acc.y = fmaf(wi, v.y, acc.y); acc.z = fmaf(wi, v.z, acc.z); acc.w = fmaf(wi, v.w, acc.w);
        }
    }
    const int status = __ldcg(&g_decode_q8_status[0]);         // looked at before the results are written
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
    *reinterpret_cast<float4*>(&s_o[warp][lane * 4]) = acc;
    __syncthreads();
    if (threadIdx.x >= 128 || status == ESP_ERR_DEVICE_TIMEOUT) return;       // of a stage 1 that gave up, partials are missing
    float M = s_m[0];
#pragma unroll
    for (int w = 1; w < W; ++w) M = fmaxf(M, s_m[w]);
    const float Mu = M == -INFINITY ? 0.f : M;
    float L = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const float f = exp2f((s_m[w] - Mu) * kLog2eQ8);
        L += s_l[w] * f;
        x += s_o[w][threadIdx.x] * f;
    }
    store_as(o, (int64_t)pair * 128 + threadIdx.x, L == 0.f ? 0.f : x / L, o_dtype);
    if (threadIdx.x == 0) lse[pair] = L == 0.f ? -INFINITY : Mu + log2f(L) * kLn2Q8;
}

int set_decode_q8_wait_limit(long long cycles) {
    ESP_CUDA_TRY(cudaMemcpyToSymbol(g_decode_q8_wait_limit_cycles, &cycles, sizeof(cycles)));
    return ESP_OK;
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

namespace esp {

template <int CODE, int GT>
static int launch_stage1_q8(DecodeQ8Args& a, cudaStream_t s) {
    // Neighbouring kv heads to a CTA, four or two where they divide evenly and lie next to each other, as long as every SM gets a CTA;
    // else one, whose tokens the four warps share.  4 requests x 512 tokens x 32 kv heads: 11.9 us with four heads, 14.8 with one;
    // 4 x 1000 x 8 kv heads: 14.2 and 12.0.
    const bool dense = a.group <= kQ8HeadTile && a.k_stride_h == 128 && a.v_stride_h == 128;
    const int64_t tiles = (int64_t)a.num_blocks * a.batch * a.head_tiles;
    if (tiles > 2147483647LL - 65536) return ESP_ERR_TOO_LARGE;
    const int nh = dense && a.head_tiles % 4 == 0 && tiles >= 4 * kNumSMs ? 4 : (dense && a.head_tiles % 2 == 0 && tiles >= 2 * kNumSMs ? 2 : 1);
    a.head_groups = a.head_tiles / nh;
    a.scale_vec = aligned16(a.k_scale) && aligned16(a.v_scale) && a.ks_stride_t % 4 == 0 && a.vs_stride_t % 4 == 0;
    const int64_t resident = kQ8Resident;
    int64_t items = tiles / nh;
    a.ranges = 0;
    if (a.parts != nullptr) {
        const int per_step = 16 * (kQ8Warps / nh);
        a.min_units = kQ8MinPiece / per_step;
        a.ranges = (int)std::max<int64_t>(1, std::min(resident / a.head_groups, (a.batch * (int64_t)a.max_len + kQ8MinPiece - 1) / kQ8MinPiece));
        items = (int64_t)a.ranges * a.head_groups;
    }
    a.counted = a.ranges > 0 || (items > resident && a.batch <= kQ8MaxCounted && !a.direct);
    const dim3 grid((unsigned)(items < resident ? items : resident));
#define ESP_S1Q(NH)                                                                                                               \
    {                                                                                                                            \
        ESP_CUDA_TRY(cudaFuncSetAttribute(decode_stage1_q8_kernel<CODE, NH, GT>, cudaFuncAttributeMaxDynamicSharedMemorySize, RingQ8<NH>::kSmem)); \
        ESP_CUDA_TRY(launch_early(decode_stage1_q8_kernel<CODE, NH, GT>, grid, kQ8Warps * 32 + 32, RingQ8<NH>::kSmem, s, a));                     \
    }
    if (nh == 4) ESP_S1Q(4) else if (nh == 2) ESP_S1Q(2) else ESP_S1Q(1)
#undef ESP_S1Q
    return ESP_OK;
}

static int stage1_q8(DecodeQ8Args& a, int head_dim, int max_len, int dtype, int code, float sm_scale, cudaStream_t s) {
    if (!a.q || !a.k || !a.v || !a.k_scale || !a.v_scale || !a.req_to_tokens || !a.b_req_idx || !a.b_seqlen || a.batch < 0 ||
        a.num_q_heads <= 0 || a.num_kv_heads <= 0 || a.num_q_heads % a.num_kv_heads || (a.seq_block_size <= 0 && !a.parts) || a.rtt_rows <= 0 ||
        a.rtt_cols <= 0 || a.pool_rows <= 0)
        return ESP_ERR_BAD_ARG;
    if (dtype != ESP_DTYPE_F16 && dtype != ESP_DTYPE_BF16) return ESP_ERR_BAD_ARG;
    if (code != ESP_CODE_INT8 && code != ESP_CODE_E4M3) return ESP_ERR_BAD_ARG;
    if (head_dim != 128) return ESP_ERR_UNSUPPORTED;
    if (a.batch > 65535 || a.num_q_heads > 65535) return ESP_ERR_TOO_LARGE;
    if (!aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || a.k_stride_t % 16 || a.k_stride_h % 16 || a.v_stride_t % 16 ||
        a.v_stride_h % 16 || ((uintptr_t)a.k_scale & 3u) || ((uintptr_t)a.v_scale & 3u))
        return ESP_ERR_ALIGNMENT;
    const int64_t nblk = (max_len + (int64_t)a.seq_block_size - 1) / a.seq_block_size;
    if (a.parts && (a.batch > kQ8MaxCounted || (max_len / 16 + 1) * (int64_t)a.batch > 2147483647LL - 65536)) return ESP_ERR_TOO_LARGE;
    a.num_blocks = (int)nblk;
    a.max_len = max_len;
    if (nblk * a.seq_block_size > 2147483647LL - 65536) return ESP_ERR_TOO_LARGE;
    a.group = a.num_q_heads / a.num_kv_heads;
    a.head_tiles = a.num_kv_heads * ((a.group + kQ8HeadTile - 1) / kQ8HeadTile);
    a.scale_log2 = (sm_scale > 0.f ? sm_scale : 1.0f / sqrtf((float)head_dim)) * kLog2eQ8;
    a.q_bf16 = dtype == ESP_DTYPE_BF16;
    if (code == ESP_CODE_INT8) return a.group <= 4 ? launch_stage1_q8<ESP_CODE_INT8, 4>(a, s) : launch_stage1_q8<ESP_CODE_INT8, 8>(a, s);
    return a.group <= 4 ? launch_stage1_q8<ESP_CODE_E4M3, 4>(a, s) : launch_stage1_q8<ESP_CODE_E4M3, 8>(a, s);
}

static DecodeQ8Args args_q8(const void* q, const void* k, const void* v, const float* k_scale, const float* v_scale, int64_t k_stride_t,
                            int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h, int64_t k_scale_stride_t, int64_t v_scale_stride_t,
                            const int32_t* req_to_tokens, int64_t req_to_tokens_stride, int32_t req_rows, int32_t req_cols,
                            const int32_t* b_req_idx, const int32_t* b_seqlen, int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                            int64_t pool_rows) {
    DecodeQ8Args a{};
    a.q = q; a.k = (const uint8_t*)k; a.v = (const uint8_t*)v; a.k_scale = k_scale; a.v_scale = v_scale;
    a.k_stride_t = k_stride_t; a.k_stride_h = k_stride_h; a.v_stride_t = v_stride_t; a.v_stride_h = v_stride_h;
    a.ks_stride_t = k_scale_stride_t; a.vs_stride_t = v_scale_stride_t;
    a.req_to_tokens = req_to_tokens; a.rtt_stride = req_to_tokens_stride; a.rtt_rows = req_rows; a.rtt_cols = req_cols;
    a.b_req_idx = b_req_idx; a.b_seqlen = b_seqlen; a.batch = batch; a.num_q_heads = num_q_heads; a.num_kv_heads = num_kv_heads;
    a.pool_rows = pool_rows;
    return a;
}

}  // namespace esp

extern "C" int esp_decode_stage1_q8(float* mid_o, float* mid_lse, const void* q, const void* k, const void* v, const float* k_scale,
                                    const float* v_scale, int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h,
                                    int64_t k_scale_stride_t, int64_t v_scale_stride_t, const int32_t* req_to_tokens,
                                    int64_t req_to_tokens_stride, int32_t req_rows, int32_t req_cols, const int32_t* b_req_idx,
                                    const int32_t* b_seqlen, int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                    int32_t max_len_in_batch, int32_t seq_block_size, int32_t dtype, int32_t code, float sm_scale,
                                    int64_t pool_rows, void* stream) {
    if (batch == 0 || max_len_in_batch <= 0) return ESP_OK;
    if (!mid_o || !mid_lse) return ESP_ERR_BAD_ARG;
    if (!aligned16(mid_o) || ((uintptr_t)mid_lse & 3u)) return ESP_ERR_ALIGNMENT;
    DecodeQ8Args a = args_q8(q, k, v, k_scale, v_scale, k_stride_t, k_stride_h, v_stride_t, v_stride_h, k_scale_stride_t, v_scale_stride_t,
                             req_to_tokens, req_to_tokens_stride, req_rows, req_cols, b_req_idx, b_seqlen, batch, num_q_heads, num_kv_heads,
                             pool_rows);
    a.mid_o = mid_o; a.mid_lse = mid_lse; a.seq_block_size = seq_block_size;
    return stage1_q8(a, head_dim, max_len_in_batch, dtype, code, sm_scale, (cudaStream_t)stream);
}

extern "C" int esp_decode_attention_q8(void* o, float* lse, float* workspace, const void* q, const void* k, const void* v,
                                       const float* k_scale, const float* v_scale, int64_t k_stride_t, int64_t k_stride_h,
                                       int64_t v_stride_t, int64_t v_stride_h, int64_t k_scale_stride_t, int64_t v_scale_stride_t,
                                       const int32_t* req_to_tokens, int64_t req_to_tokens_stride, int32_t req_rows, int32_t req_cols,
                                       const int32_t* b_req_idx, const int32_t* b_seqlen, int32_t batch, int32_t num_q_heads,
                                       int32_t num_kv_heads, int32_t head_dim, int32_t max_len_in_batch, int32_t seq_block_size,
                                       int32_t dtype, int32_t o_dtype, int32_t code, float sm_scale, int64_t pool_rows, void* stream) {
    if (batch == 0) return ESP_OK;
    if (!o || !lse || max_len_in_batch < 0 || seq_block_size < 0 || num_q_heads <= 0) return ESP_ERR_BAD_ARG;
    if (o_dtype != ESP_DTYPE_F16 && o_dtype != ESP_DTYPE_BF16 && o_dtype != ESP_DTYPE_F32) return ESP_ERR_BAD_ARG;
    const int32_t max_len = max_len_in_batch > 0 ? max_len_in_batch : 1;
    // seq_block_size 0: equal pieces, or one split where no request is longer than 256 tokens (512 from 8 requests on), which saves
    // the merge.  Pieces / one split in us, 8 kv heads, group 4: one request of 256 tokens 8.7 / 7.4; 16 of 512 11.7 / 11.2, 64 of
    // them 25.6 / 20.5, 256 71.4 / 65.3; 32 kv heads, 8 of 512 16.4 / 14.3.  The rule does not count heads: with a single kv head there are
    // too few CTAs in one split (8 requests of 512 tokens 9.4 / 10.8, 32 of them 10.1 / 11.1).
    const bool even = seq_block_size == 0 && max_len > q8_whole(batch);
    const int32_t block = seq_block_size == 0 ? (even ? kQ8MinPiece : max_len) : seq_block_size;
    const int64_t nblk = (max_len + (int64_t)block - 1) / block;
    if (nblk > 1 && !workspace) return ESP_ERR_BAD_ARG;
    if (!aligned16(o) || ((uintptr_t)lse & 3u) || (nblk > 1 && !aligned16(workspace))) return ESP_ERR_ALIGNMENT;
    DecodeQ8Args a = args_q8(q, k, v, k_scale, v_scale, k_stride_t, k_stride_h, v_stride_t, v_stride_h, k_scale_stride_t, v_scale_stride_t,
                             req_to_tokens, req_to_tokens_stride, req_rows, req_cols, b_req_idx, b_seqlen, batch, num_q_heads, num_kv_heads,
                             pool_rows);
    const int64_t rows = even ? (std::min<int64_t>(kQ8Resident, (batch * (int64_t)max_len + kQ8MinPiece - 1) / kQ8MinPiece) + batch) * num_q_heads
                              : nblk * batch * num_q_heads;
    a.mid_o = workspace; a.mid_lse = workspace + rows * 128; a.seq_block_size = block;
    a.o = o; a.lse = lse; a.o_dtype = o_dtype; a.direct = nblk == 1;
    if (even) a.parts = reinterpret_cast<int*>(workspace + rows * 129);
    cudaStream_t s = (cudaStream_t)stream;
    const int rc = stage1_q8(a, head_dim, max_len, dtype, code, sm_scale, s);
    if (rc || nblk == 1) return rc;
    const unsigned pairs = (unsigned)((int64_t)batch * num_q_heads);
    // splits of one request, on average
    const bool wide = (even ? a.ranges / batch : nblk) > 64;
    ESP_CUDA_TRY(launch_early(wide ? decode_merge_q8_kernel<16> : decode_merge_q8_kernel<4>, dim3(pairs), wide ? 512 : 128, 0, s, o, lse, b_seqlen,
                              a.mid_o, a.mid_lse, a.parts, batch, num_q_heads, (int)nblk, block, o_dtype));
    return ESP_OK;
}
