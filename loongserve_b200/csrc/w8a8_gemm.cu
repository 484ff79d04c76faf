// Product of 8-bit integer matrices with a scale for every token and every output channel:
//   out[m, n] = (sum_k a[m, k] * w[n, k]) * a_scale[m] * w_scale[n]
// a [M, K] int8 rows of tokens, w [N, K] int8 rows of output channels (both with K contiguous), 32-bit integer sums in tensor
// memory (tcgen05.mma kind::i8); in the epilogue the sum becomes fp32 (rounded where it has more than 24 bits), is multiplied twice and
// rounded to the output type.  K <= 131071 keeps every
// sum inside 32 bits (128 * 128 * K < 2^31).  Integer sums do not depend on their order, so every split below gives the same bits.
//
// Operand tiles are 128 bytes of K wide, 128-byte swizzle, fetched by TMA (rows and bytes behind the matrix arrive as zeros).
#include <cuda.h>

#include "quant_common.cuh"
#include "sm100_ptx.cuh"

namespace esp {

using namespace ptx;

constexpr int kBK = 128;                 // bytes of K per stage: one swizzle row, four MMA steps of 32

// Status of the bounded mbarrier waits: {ESP_ERR_DEVICE_TIMEOUT, block, which wait, detail}; their limit in SM cycles.
__device__ int g_mm_status[4];
__device__ long long g_mm_wait_limit_cycles = 2000000000LL;

enum MmWait { MW_EMPTY = 100, MW_FULL = 101, MW_ACC_EMPTY = 102, MW_ACC_FULL = 103, MW_DRAIN = 104 };

__device__ __noinline__ void mm_timeout(int which, int detail) {
    if (atomicCAS(&g_mm_status[0], 0, ESP_ERR_DEVICE_TIMEOUT) == 0) {
        g_mm_status[1] = blockIdx.x + gridDim.x * blockIdx.y;
        g_mm_status[2] = which;
        g_mm_status[3] = detail;
    }
}
// false: the wait ran out (here or, through *s_abort, in another warp of the CTA); the caller drains and leaves
__device__ __forceinline__ bool mm_wait(uint32_t bar, uint32_t parity, volatile int* s_abort, int which, int detail) {
    const int r = mbar_wait_bounded(bar, parity, &g_mm_wait_limit_cycles, s_abort);
    if (r == 2) { mm_timeout(which, detail); *s_abort = 1; }
    return r == 0;
}
// after an abort: wait (bounded, whatever the abort flag says) for work of one's own that is still in flight
__device__ __forceinline__ void mm_drain(uint32_t bar, uint32_t parity) {
    mbar_wait_bounded(bar, parity, &kDrainLimitCycles, nullptr);
}

template <typename OT> __device__ __forceinline__ OT from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename OT> struct Pack16;      // 16 bytes of outputs from consecutive fp32 values
template <> struct Pack16<float> {
    static constexpr int n = 4;
    static __device__ __forceinline__ uint4 go(const float* x) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
};
template <typename OT> struct Pack16 {
    static constexpr int n = 8;
    static __device__ __forceinline__ uint4 go(const float* x) {
        return make_uint4(Cvt<OT>::pack(x[0], x[1]), Cvt<OT>::pack(x[2], x[3]), Cvt<OT>::pack(x[4], x[5]), Cvt<OT>::pack(x[6], x[7]));
    }
};

struct MmArgs {
    void* out; int64_t ldo; const float* a_scale; const float* w_scale;
    int64_t M, N; int kstages;           // kstages = ceil(K / 128)
    int m_tiles, n_tiles;
    int vec_out;                         // rows of out are 16-byte aligned
};

// ------------------------------------------------------------------------------------------------
// Many tokens: CTA pairs (cluster of two, cta_group::2).  A pair owns 256 tokens x PN channels; CTA c holds 128 of the tokens
// (A) and half of the channels (B), one thread of the even CTA issues the M = 256 MMAs that run on both SMs.  Persistent: each
// pair walks over tiles; two accumulators of PN columns take turns, so the epilogue of one tile runs under the next one's MMAs.
// Warps: 0 producer, 1 issuer (and tensor-memory owner), 2-3 idle, 4-7 epilogue (one token row per thread).
constexpr int kPairM = 128, kPairThreads = 256;
constexpr int kEpiRowBytes = 128 + 16;                                           // one staged row piece, padded against bank conflicts
template <int PN> struct Pair {
    static constexpr int kStages = PN == 256 ? 6 : 8;
    static constexpr int kStageBytes = kPairM * kBK + PN / 2 * kBK;              // 32 or 24 KiB per CTA
    static constexpr int kOffEpi = kStages * kStageBytes;                        // per epilogue warp: 32 row pieces, PN channel scales
    static constexpr int kEpiWarp = 32 * kEpiRowBytes + PN * 4;
    static constexpr int kOffBar = kOffEpi + 4 * kEpiWarp;
    static constexpr int kFull = 0, kEmpty = kStages, kAccFull = 2 * kStages, kAccEmpty = 2 * kStages + 2, kDrain = 2 * kStages + 4, kBars = 2 * kStages + 5;
    static constexpr int kOffMisc = kOffBar + kBars * 8;
    static constexpr int kSmem = kOffMisc + 32 + 1024;
};
static_assert(Pair<256>::kSmem <= 232448 && Pair<128>::kSmem <= 232448, "shared memory of one CTA");

// Tiles are walked in bands of 8 token tiles: the pairs that run together share both operands' tiles in L2.
__device__ __forceinline__ void tile_of(int t, int m_tiles, int n_tiles, int& m, int& n) {
    constexpr int kBand = 8;
    const int band = t / (kBand * n_tiles), in_band = t - band * kBand * n_tiles;
    const int rows = min(kBand, m_tiles - band * kBand);
    n = in_band / rows;
    m = band * kBand + (in_band - n * rows);
}

// After a wait ran out: neither CTA may leave while MMAs or copies of either are under way, because copies write the CTA that started
// them and count on the even CTA's barriers.  The two may have come a different number of steps far (issued, peer_issued): a step
// that one of them alone has started is made to expect that CTA's bytes alone.  The issuing thread has committed kDrain.
template <int PN>
__device__ __noinline__ void pair_drain(uint32_t base, uint32_t cta, int issued, int peer_issued) {
    using C = Pair<PN>;
    auto bar = [base](int i) { return base + C::kOffBar + 8u * i; };
    if (threadIdx.x == 32) mm_drain(bar(C::kDrain), 0);
    if (cta == 0 && threadIdx.x == 0) {
        const int hi = max(issued, peer_issued);
        for (int i = max(hi - C::kStages, 0); i < hi; ++i) {
            const uint32_t b = bar(C::kFull + i % C::kStages);
            if (i >= issued) mbar_expect_tx(b, C::kStageBytes);
            else if (i >= peer_issued) mbar_complete_tx(b, C::kStageBytes);
            mm_drain(b, (i / C::kStages) & 1);
        }
    }
}

template <typename OT, int PN>
__global__ void __launch_bounds__(kPairThreads, 1) mm_w8a8_pair_kernel(const __grid_constant__ CUtensorMap tm_a,
                                                                       const __grid_constant__ CUtensorMap tm_w, const MmArgs p) {
    using C = Pair<PN>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    auto bar = [base](int i) { return base + C::kOffBar + 8u * i; };
    auto lbar = [&bar](int i) { return map_to_cta(bar(i), 0u); };               // the even CTA's barrier
    volatile uint32_t* s_tmem = reinterpret_cast<volatile uint32_t*>(gen + C::kOffMisc);
    volatile int* s_abort = reinterpret_cast<volatile int*>(gen + C::kOffMisc + 4);
    volatile int* s_issued = reinterpret_cast<volatile int*>(gen + C::kOffMisc + 8);     // steps whose copies this CTA has started
    volatile int* s_peer = reinterpret_cast<volatile int*>(gen + C::kOffMisc + 16);      // the other CTA's s_abort and s_issued, at the end
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t cta = cluster_ctarank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int tiles = p.m_tiles * p.n_tiles;

    if (threadIdx.x == 0) {
        *s_abort = (*reinterpret_cast<volatile int*>(&g_mm_status[0]) != 0) ? 1 : 0;    // after a reported timeout nothing is started
        *s_issued = 0;
        for (int i = 0; i < C::kBars; ++i) mbar_init(bar(i), (i == C::kAccEmpty || i == C::kAccEmpty + 1) ? 8 : 1);
        fence_barrier_init();
        prefetch_tensormap(&tm_a); prefetch_tensormap(&tm_w);
    }
    __syncthreads();
    if (warp == 1) { tmem_alloc_pair(base + C::kOffMisc, 2 * PN); tmem_relinquish_pair(); }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;

    if (warp == 0) {
        if (lane == 0 && !*s_abort) {
            int it = 0;
            bool ok = true;
            for (int t = pair; t < tiles && ok; t += pairs) {
                int mt, nt;
                tile_of(t, p.m_tiles, p.n_tiles, mt, nt);
                const int m0 = mt * 2 * kPairM + (int)cta * kPairM, n0 = nt * PN + (int)cta * (PN / 2);
                for (int k = 0; k < p.kstages; ++k, ++it) {
                    const int st = it % C::kStages;
                    if (it >= C::kStages && !(ok = mm_wait(bar(C::kEmpty + st), ((it / C::kStages) - 1) & 1, s_abort, MW_EMPTY, it))) break;
                    if (cta == 0) mbar_expect_tx(bar(C::kFull + st), 2 * C::kStageBytes);
                    const uint32_t dst = base + st * C::kStageBytes;
                    tma_load_2d_pair(dst, &tm_a, lbar(C::kFull + st), k * kBK, m0);
                    tma_load_2d_pair(dst + kPairM * kBK, &tm_w, lbar(C::kFull + st), k * kBK, n0);
                }
            }
            // A look at the last steps, a millisecond each at most; what is still under way then is waited for at the end.  (Measured: with
            // the loop above alone the compiler makes something of it that takes 1002 us instead of 995 for 16384 x 22016 x 4096.)
            if (!ok && cta == 0)
                for (int i = it > C::kStages ? it - C::kStages : 0; i < it; ++i) mbar_try_wait(bar(C::kFull + i % C::kStages), (i / C::kStages) & 1);
            *s_issued = it;
        }
    } else if (warp == 1) {
        if (cta == 0 && lane == 0 && !*s_abort) {
            constexpr uint32_t idesc = make_idesc_i8(2 * kPairM, PN);
            int it = 0, n_tile = 0;
            bool ok = true;
            for (int t = pair; t < tiles && ok; t += pairs, ++n_tile) {
                const int buf = n_tile & 1;
                if (n_tile >= 2 && !(ok = mm_wait(bar(C::kAccEmpty + buf), ((n_tile >> 1) - 1) & 1, s_abort, MW_ACC_EMPTY, n_tile))) break;
                tc_fence_after();
                for (int k = 0; k < p.kstages; ++k, ++it) {
                    const int st = it % C::kStages;
                    if (!(ok = mm_wait(bar(C::kFull + st), (it / C::kStages) & 1, s_abort, MW_FULL, it))) break;
                    tc_fence_after();
                    const uint32_t sa = base + st * C::kStageBytes, sb = sa + kPairM * kBK;
#pragma unroll
                    for (int j = 0; j < kBK / 32; ++j)
                        umma_i8_pair_ss(tmem + buf * PN, desc_kmajor_sw128(sa + j * 32), desc_kmajor_sw128(sb + j * 32), idesc, (k | j) != 0);
                    umma_pair_commit(bar(C::kEmpty + st));
                }
                if (ok) umma_pair_commit(bar(C::kAccFull + buf));
            }
        }
    } else if (warp >= 4) {
        const int w = warp - 4;
        uint8_t* stage = gen + C::kOffEpi + w * C::kEpiWarp;
        float* sw = reinterpret_cast<float*>(stage + 32 * kEpiRowBytes);
        constexpr int kCols = 128 / (int)sizeof(OT);           // channels per staged piece (128 bytes of a row)
        OT* out = reinterpret_cast<OT*>(p.out);
        bool ok = !*s_abort;
        int n_tile = 0;
        for (int t = pair; t < tiles && ok; t += pairs, ++n_tile) {
            int mt, nt;
            tile_of(t, p.m_tiles, p.n_tiles, mt, nt);
            const int64_t row0 = (int64_t)mt * 2 * kPairM + (int64_t)cta * kPairM + w * 32;      // first row of this warp
            const int64_t n0 = (int64_t)nt * PN;
            const int buf = n_tile & 1;
            __syncwarp();
            for (int i = lane; i < PN; i += 32) sw[i] = n0 + i < p.N ? p.w_scale[n0 + i] : 0.f;
            const float sa = row0 + lane < p.M ? p.a_scale[row0 + lane] : 0.f;
            ok = mm_wait(bar(C::kAccFull + buf), (n_tile >> 1) & 1, s_abort, MW_ACC_FULL, n_tile);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint32_t acc = tmem + buf * PN + ((uint32_t)(w * 32) << 16);
            const int rows = (int)min((int64_t)32, p.M - row0);
#pragma unroll 1
            for (int c0 = 0; c0 < PN; c0 += kCols) {
                uint32_t r[kCols / 32][32];
#pragma unroll
                for (int h = 0; h < kCols / 32; ++h) tmem_ld32(acc + c0 + h * 32, r[h]);
                tmem_wait_ld();
                if (c0 + kCols == PN) {                     // the last read of this accumulator: the issuer may have it back
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(lbar(C::kAccEmpty + buf));
                }
#pragma unroll
                for (int h = 0; h < kCols / 32; ++h)
#pragma unroll
                    for (int i = 0; i < 32; i += Pack16<OT>::n) {
                        float x[Pack16<OT>::n];
#pragma unroll
                        for (int j = 0; j < Pack16<OT>::n; ++j) x[j] = __int2float_rn((int)r[h][i + j]) * sa * sw[c0 + h * 32 + i + j];
                        *reinterpret_cast<uint4*>(stage + lane * kEpiRowBytes + (h * 32 + i) * (int)sizeof(OT)) = Pack16<OT>::go(x);
                    }
                __syncwarp();
                const int64_t nleft = p.N - n0 - c0;
                const int ncols = nleft < kCols ? (int)nleft : kCols;
                if (p.vec_out) {
                    const int c16 = (lane & 7) * Pack16<OT>::n;             // 4 rows of 128 bytes per step, 16 bytes per lane
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int rr = i * 4 + (lane >> 3);
                        if (rr >= rows || c16 >= ncols) continue;
                        const uint8_t* from = stage + rr * kEpiRowBytes + (lane & 7) * 16;
                        OT* to = out + (row0 + rr) * p.ldo + n0 + c0 + c16;
                        if (c16 + Pack16<OT>::n <= ncols) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
                        else
                            for (int j = 0; j < ncols - c16; ++j) to[j] = reinterpret_cast<const OT*>(from)[j];
                    }
                } else {
                    for (int i = lane; i < ncols; i += 32) {
#pragma unroll 8
                        for (int rr = 0; rr < rows; ++rr)
                            out[(row0 + rr) * p.ldo + n0 + c0 + i] = *reinterpret_cast<const OT*>(stage + rr * kEpiRowBytes + i * sizeof(OT));
                    }
                }
                __syncwarp();
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0) {
        st_cluster_u32(map_to_cta(base + C::kOffMisc + 16, cta ^ 1u), (uint32_t)*s_abort);
        st_cluster_u32(map_to_cta(base + C::kOffMisc + 20, cta ^ 1u), (uint32_t)*s_issued);
    }
    cluster_sync_all();                  // neither CTA frees tensor memory while the peer's MMAs may still use it
    if (*s_abort | s_peer[0]) {          // a wait ran out in one of the CTAs: both see it here
        if (threadIdx.x == 32 && cta == 0) umma_pair_commit(bar(C::kDrain));
        pair_drain<PN>(base, cta, *s_issued, s_peer[1]);
        __syncthreads();
        cluster_sync_all();
    }
    if (warp == 1) { tc_fence_after(); tmem_dealloc_pair(tmem, 2 * PN); }
}

// ------------------------------------------------------------------------------------------------
// Few tokens: the weights are what is read, so channels take the 128 rows of the MMA and TN tokens its columns.  A cluster of S
// CTAs splits K of one tile; the integer partials are summed through distributed shared memory (each CTA sums and writes TN / S
// of the tokens).  Warps: 0 producer, 1 issuer, 2-5 epilogue (one channel per thread).
//
// Some 6 us of such a call are not its bytes, so its start (barriers, tensor memory, descriptors) runs under the kernel before it
// where that one allows it (the row kernels, this one): nothing of that kernel's results is touched before grid_dependency_wait, and
// after it only by loads that pass the L1; the scales wait in shared memory for the sums.  One after the other (us, tokens x
// channels x K): 64 x 4096 x 4096 10.6 -> 8.9, 1 x 22016 x 4096 19.5 -> 17.6, 64 x 4096 x 11008 14.5 -> 13.4; norm, product, SiLU and
// product of a layer of 4096 and 11008: 37.5 -> 33.9 for one token, 46.2 -> 43.0 for 64.
constexpr int kSkinnyThreads = 192;
template <int TN> struct Skinny {
    static_assert(TN == 16 || TN == 32 || TN == 64 || TN == 128, "tokens of a tile");
    static constexpr int kStageBytes = 128 * kBK + TN * kBK;
    static constexpr int kStages = TN >= 128 ? 3 : (TN >= 64 ? 4 : 5);      // two CTAs to an SM
    static constexpr int kDump = 128 * TN * 4;                      // partials, over the pipeline's stages once they are used up
    static constexpr int kBody = kStages * kStageBytes > kDump ? kStages * kStageBytes : kDump;
    static constexpr int kOffBar = kBody;
    static constexpr int kOffMisc = kOffBar + (2 * kStages + 1) * 8;
    static constexpr int kOffScale = kOffMisc + 16;                 // of the tile's tokens, of its channels
    static constexpr int kSmem = kOffScale + (TN + 128) * 4 + 1024;
    static constexpr int kCols = TN < 32 ? 32 : TN;
};

template <typename OT, int TN>
__global__ void __launch_bounds__(kSkinnyThreads) mm_w8a8_skinny_kernel(const __grid_constant__ CUtensorMap tm_a,
                                                                        const __grid_constant__ CUtensorMap tm_w, const MmArgs p, int splits) {
    using C = Skinny<TN>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    auto bar = [base](int i) { return base + C::kOffBar + 8u * i; };      // full [stages], empty [stages], done
    volatile uint32_t* s_tmem = reinterpret_cast<volatile uint32_t*>(gen + C::kOffMisc);
    volatile int* s_abort = reinterpret_cast<volatile int*>(gen + C::kOffMisc + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = (int)cluster_ctarank();
    const int n0 = (blockIdx.x / splits) * 128, m0 = blockIdx.y * TN;
    const int k0 = (int)((int64_t)p.kstages * split / splits), k1 = (int)((int64_t)p.kstages * (split + 1) / splits);
    const int nk = k1 - k0;                                               // at least one: splits <= kstages

    if (threadIdx.x == 0) {
        *s_abort = (*reinterpret_cast<volatile int*>(&g_mm_status[0]) != 0) ? 1 : 0;
        for (int i = 0; i < 2 * C::kStages + 1; ++i) mbar_init(bar(i), 1);
        fence_barrier_init();
        prefetch_tensormap(&tm_a); prefetch_tensormap(&tm_w);
    }
    if (warp == 1) { tmem_alloc(base + C::kOffMisc, C::kCols); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    if (splits > 1) cluster_arrive();                                     // s_abort is set up: the other CTAs may write it
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    grid_dependency_wait();
    grid_dependents_launch();
    bool ok = !*s_abort;

    if (warp == 0) {
        if (lane == 0 && ok) {
            int it = 0;
            for (; it < nk; ++it) {
                const int st = it % C::kStages;
                if (it >= C::kStages && !(ok = mm_wait(bar(C::kStages + st), ((it / C::kStages) - 1) & 1, s_abort, MW_EMPTY, it))) break;
                mbar_expect_tx(bar(st), C::kStageBytes);
                const uint32_t dst = base + st * C::kStageBytes;
                tma_load_2d(dst, &tm_w, bar(st), (k0 + it) * kBK, n0);
                tma_load_2d(dst + 128 * kBK, &tm_a, bar(st), (k0 + it) * kBK, m0);
            }
            // whichever warp gives up, the CTA does not leave before the copies have landed
            for (int i = it > C::kStages ? it - C::kStages : 0; i < it; ++i) mm_drain(bar(i % C::kStages), (i / C::kStages) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0 && ok) {
            constexpr uint32_t idesc = make_idesc_i8(128, TN);
            for (int it = 0; it < nk; ++it) {
                const int st = it % C::kStages;
                if (!(ok = mm_wait(bar(st), (it / C::kStages) & 1, s_abort, MW_FULL, it))) break;
                tc_fence_after();
                const uint32_t sw = base + st * C::kStageBytes, sa = sw + 128 * kBK;
#pragma unroll
                for (int j = 0; j < kBK / 32; ++j)
                    umma_i8_ss(tmem, desc_kmajor_sw128(sw + j * 32), desc_kmajor_sw128(sa + j * 32), idesc, (it | j) != 0);
                umma_commit(bar(C::kStages + st));
            }
            umma_commit(bar(2 * C::kStages));                             // every MMA issued, in the aborted case too
            if (!ok) mm_drain(bar(2 * C::kStages), 0);
        }
    }
    int32_t* dump = reinterpret_cast<int32_t*>(gen);                      // [TN][128]
    float* s_scale = reinterpret_cast<float*>(gen + C::kOffScale);
    if (warp >= 2) {
        for (int i = threadIdx.x - 64; i < TN + 128; i += 128) {          // while the MMAs run
            const int64_t at = i < TN ? m0 + i : n0 + (i - TN);
            s_scale[i] = at < (i < TN ? p.M : p.N) ? __ldcg((i < TN ? p.a_scale : p.w_scale) + at) : 0.f;
        }
        const int q = warp & 3;                                           // the quarter of the tensor-memory lanes this warp may read
        if (ok) ok = mm_wait(bar(2 * C::kStages), 0, s_abort, MW_DRAIN, nk);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < TN; c += 16) {
                uint32_t r[16];
                tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + c, r);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) dump[(c + i) * 128 + q * 32 + lane] = (int)r[i];
            }
            tc_fence_before();
        }
    }
    // Every CTA of the cluster passes here.  One whose waits ran out has no partials: it tells the others, and nothing is written.
    __syncthreads();
    if (splits > 1) {
        cluster_wait();
        if (threadIdx.x < splits && *s_abort) st_cluster_u32(map_to_cta(base + C::kOffMisc + 4, threadIdx.x), 1u);
        cluster_sync_all();
    }
    if (!*s_abort) {
        OT* out = reinterpret_cast<OT*>(p.out);
        const int t_lo = TN * split / splits, t_hi = TN * (split + 1) / splits;
        const int64_t M = p.M, N = p.N;
        const uint32_t my = base;
        for (int i = threadIdx.x; i < (t_hi - t_lo) * 64; i += kSkinnyThreads) {       // two channels of one token
            const int t = t_lo + (i >> 6), ch = (i & 63) * 2;
            const int64_t m = m0 + t, n = n0 + ch;
            if (m >= M) break;
            if (n >= N) continue;
            int s0 = 0, s1 = 0;
            for (int r = 0; r < splits; ++r) {
                int v0, v1;
                const uint32_t at = (splits > 1 ? map_to_cta(my, r) : my) + (uint32_t)(t * 128 + ch) * 4u;
                asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];" : "=r"(v0), "=r"(v1) : "r"(at));
                s0 += v0; s1 += v1;
            }
            const float sa = s_scale[t];
            const float x0 = __int2float_rn(s0) * sa * s_scale[TN + ch];
            OT* o = out + m * p.ldo + n;
            if (n + 1 < N) {
                const float x1 = __int2float_rn(s1) * sa * s_scale[TN + ch + 1];
                if (p.vec_out) {
                    if constexpr (sizeof(OT) == 2) *reinterpret_cast<uint32_t*>(o) = Cvt<OT>::pack(x0, x1);
                    else *reinterpret_cast<float2*>(o) = make_float2(x0, x1);
                } else { o[0] = from_f32<OT>(x0); o[1] = from_f32<OT>(x1); }
            } else {
                o[0] = from_f32<OT>(x0);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (splits > 1) cluster_sync_all();                                   // peers may still read this CTA's partials
    if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem, C::kCols); }
}

// ------------------------------------------------------------------------------------------------
typedef CUresult (*MmEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// int8 matrix [rows, K]: box = 128 bytes of K x box_rows rows, 128-byte swizzle
static int make_map(CUtensorMap* tm, const int8_t* p, int64_t rows, int64_t k, int64_t ld, int box_rows) {
    static MmEncodeFn fn = nullptr;
    if (!fn) {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<MmEncodeFn>(f);
        if (!fn) { snprintf(last_cuda_error_buf(), 256, "cuTensorMapEncodeTiled entry point not found"); return ESP_ERR_CUDA; }
    }
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {(cuuint32_t)kBK, (cuuint32_t)box_rows}, es[2] = {1, 1};
    const CUresult r = fn(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        snprintf(last_cuda_error_buf(), 256, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
        return ESP_ERR_CUDA;
    }
    return ESP_OK;
}

constexpr int kMaxMmDevices = 64;

// How many CTA pairs the device keeps resident at once (asked once per device and kernel).
template <typename OT, int PN>
static int resident_pairs(int* out) {
    static int known[kMaxMmDevices] = {0};
    int dev = -1;
    ESP_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= kMaxMmDevices) return ESP_ERR_UNSUPPORTED;
    if (!known[dev]) {
        ESP_CUDA_TRY(cudaFuncSetAttribute(mm_w8a8_pair_kernel<OT, PN>, cudaFuncAttributeMaxDynamicSharedMemorySize, Pair<PN>::kSmem));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(kNumSMs / 2 * 2); cfg.blockDim = dim3(kPairThreads); cfg.dynamicSmemBytes = Pair<PN>::kSmem;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = 2; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
        cfg.attrs = at; cfg.numAttrs = 1;
        int n = 0;
        ESP_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, mm_w8a8_pair_kernel<OT, PN>, &cfg));
        known[dev] = n > 0 ? n : 1;
    }
    *out = known[dev];
    return ESP_OK;
}

template <typename OT, int PN>
static int launch_pair(const int8_t* a, int64_t lda, const int8_t* w, int64_t ldw, int64_t k, MmArgs g, cudaStream_t s) {
    CUtensorMap ta, tw;
    int rc = make_map(&ta, a, g.M, k, lda, kPairM);
    if (!rc) rc = make_map(&tw, w, g.N, k, ldw, PN / 2);
    int pairs = 0;
    if (!rc) rc = resident_pairs<OT, PN>(&pairs);
    if (rc) return rc;
    g.m_tiles = (int)((g.M + 2 * kPairM - 1) / (2 * kPairM));
    g.n_tiles = (int)((g.N + PN - 1) / PN);
    const int64_t tiles = (int64_t)g.m_tiles * g.n_tiles;
    if (tiles > 2147483647LL) return ESP_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (unsigned)(tiles < pairs ? tiles : pairs)); cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = Pair<PN>::kSmem; cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    ESP_CUDA_TRY(cudaFuncSetAttribute(mm_w8a8_pair_kernel<OT, PN>, cudaFuncAttributeMaxDynamicSharedMemorySize, Pair<PN>::kSmem));
    ESP_CUDA_TRY(cudaLaunchKernelEx(&cfg, mm_w8a8_pair_kernel<OT, PN>, ta, tw, g));
    return ESP_OK;
}

template <typename OT, int TN>
static int launch_skinny(const int8_t* a, int64_t lda, const int8_t* w, int64_t ldw, int64_t k, MmArgs g, int splits, cudaStream_t s) {
    using C = Skinny<TN>;
    CUtensorMap ta, tw;
    int rc = make_map(&ta, a, g.M, k, lda, TN);
    if (!rc) rc = make_map(&tw, w, g.N, k, ldw, 128);
    if (rc) return rc;
    const int64_t nt = (g.N + 127) / 128, mt = (g.M + TN - 1) / TN;
    if (mt > 65535 || nt * splits > 2147483647LL) return ESP_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(nt * splits), (unsigned)mt); cfg.blockDim = dim3(kSkinnyThreads);
    cfg.dynamicSmemBytes = C::kSmem; cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = splits; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at; cfg.numAttrs = 2;
    ESP_CUDA_TRY(cudaFuncSetAttribute(mm_w8a8_skinny_kernel<OT, TN>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    ESP_CUDA_TRY(cudaLaunchKernelEx(&cfg, mm_w8a8_skinny_kernel<OT, TN>, ta, tw, g, splits));
    return ESP_OK;
}

template <typename OT>
static int launch_mm(const int8_t* a, int64_t lda, const int8_t* w, int64_t ldw, int64_t k, MmArgs g, cudaStream_t s) {
    g.kstages = (int)((k + kBK - 1) / kBK);
    g.vec_out = ((uintptr_t)g.out % 16 == 0 && (g.ldo * (int64_t)sizeof(OT)) % 16 == 0) ? 1 : 0;
    // The variant with the least estimated time (us).  A skinny CTA costs about 6 us around its stages; a stage costs less while
    // every SM has one CTA than with two (which then share the SM's intake).  A pair costs 5.4 or 6.5 us and 0.29 or 0.31 us per
    // stage and wave of tiles.  Measured against these estimates (B200, tokens x channels x K, us,
    // each call by itself; with its start under the kernel before it a skinny one takes 1 to 2 us less, which the estimates leave out: near
    // a border pairs are taken somewhat too often):
    //   64 x 4096 x 11008: TN 64 in 8 splits 13.8, 4 splits 15.2, 1 split 29.2, pairs 31.0      256 x 4096 x 11008: TN 128 in 4 splits 20.1, pairs 31.0
    //   256 x 22016 x 4096: TN 64 50.8, TN 128 54.3, pairs of 256 29.7                          512 x 4096 x 1280: TN 64 12.9, pairs of 128 8.3, of 256 9.6
    //   600 x 600 x 8000: TN 64 in 4 splits 12.4, TN 128 in 8 splits 12.5, pairs of 128 24.6    400 x 8000 x 2992: pairs of 256 17.2, of 128 21.0, TN 128 36.7
    // Splits are powers of two: clusters of other sizes leave SMs of a GPC unused (64 x 12288 x 4096: 25.3 us in 3 splits, 17.7 in 2).
    const int64_t nt = (g.N + 127) / 128, m2 = (g.M + 255) / 256, pairs = kNumSMs / 2;
    const int ks = g.kstages;
    auto waves = [](int64_t n, int64_t per) { return (double)((n + per - 1) / per); };
    const double pair256 = 6.5 + waves(m2 * ((g.N + 255) / 256), pairs) * ks * 0.31, pair128 = 5.4 + waves(m2 * nt, pairs) * ks * 0.29;
    double best = pair256 < pair128 ? pair256 : pair128;
    int tn = 0, splits = 1;
    const int tn_first = g.M <= 16 ? 16 : (g.M <= 32 ? 32 : 64), tn_last = g.M <= 64 ? tn_first : 128;
    if (g.M <= 4096)
        for (int t = tn_first; t <= tn_last; t *= 2)
            for (int sp = 1; sp <= 8 && sp <= ks; sp *= 2) {
                const int64_t ctas = nt * ((g.M + t - 1) / t) * sp;
                const double one = t <= 32 ? 0.26 : (t == 64 ? 0.33 : 0.45), two = t <= 32 ? 0.50 : (t == 64 ? 0.62 : 0.75);
                const double est = waves(ctas, 2 * kNumSMs) * (6.0 + (ks + sp - 1) / sp * (ctas <= kNumSMs ? one : two));
                if (est < best) { best = est; tn = t; splits = sp; }
            }
    switch (tn) {
        case 16: return launch_skinny<OT, 16>(a, lda, w, ldw, k, g, splits, s);
        case 32: return launch_skinny<OT, 32>(a, lda, w, ldw, k, g, splits, s);
        case 64: return launch_skinny<OT, 64>(a, lda, w, ldw, k, g, splits, s);
        case 128: return launch_skinny<OT, 128>(a, lda, w, ldw, k, g, splits, s);
        default: break;
    }
    return pair256 <= pair128 ? launch_pair<OT, 256>(a, lda, w, ldw, k, g, s) : launch_pair<OT, 128>(a, lda, w, ldw, k, g, s);
}

int mm_w8a8_status(int32_t out[4], int32_t clear) {
    ESP_CUDA_TRY(cudaMemcpyFromSymbol(out, g_mm_status, sizeof(int) * 4));
    if (clear) {
        int zero[4] = {0, 0, 0, 0};
        ESP_CUDA_TRY(cudaMemcpyToSymbol(g_mm_status, zero, sizeof(zero)));
    }
    return ESP_OK;
}
int set_mm_wait_limit(long long cycles) {
    ESP_CUDA_TRY(cudaMemcpyToSymbol(g_mm_wait_limit_cycles, &cycles, sizeof(cycles)));
    return ESP_OK;
}

}  // namespace esp

using namespace esp;

extern "C" int esp_mm_w8a8(void* out, int64_t out_row_stride, const int8_t* a, int64_t a_row_stride, const float* a_scale, const int8_t* w,
                           int64_t w_row_stride, const float* w_scale, int64_t m, int64_t n, int64_t k, int32_t out_dtype, void* stream) {
    if (m == 0 || n == 0) return ESP_OK;
    if (!out || !a || !a_scale || !w || !w_scale || m < 0 || n < 0 || k <= 0) return ESP_ERR_BAD_ARG;
    if (out_dtype != ESP_DTYPE_F16 && out_dtype != ESP_DTYPE_BF16 && out_dtype != ESP_DTYPE_F32) return ESP_ERR_BAD_ARG;
    if (out_row_stride < n || a_row_stride < k || w_row_stride < k) return ESP_ERR_BAD_ARG;
    if (k % 16 || a_row_stride % 16 || w_row_stride % 16 || !aligned16(a) || !aligned16(w)) return ESP_ERR_ALIGNMENT;
    if (k > 131071 || m > 2147483392LL || n > 2147483392LL) return ESP_ERR_TOO_LARGE;       // tile coordinates are 32-bit
    MmArgs g{out, out_row_stride, a_scale, w_scale, m, n, 0, 0, 0, 0};
    cudaStream_t s = (cudaStream_t)stream;
    if (out_dtype == ESP_DTYPE_F16) return launch_mm<__half>(a, a_row_stride, w, w_row_stride, k, g, s);
    if (out_dtype == ESP_DTYPE_BF16) return launch_mm<__nv_bfloat16>(a, a_row_stride, w, w_row_stride, k, g, s);
    return launch_mm<float>(a, a_row_stride, w, w_row_stride, k, g, s);
}
