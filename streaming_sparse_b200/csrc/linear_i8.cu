// linear_i8.cu -- the 8-bit linear layer: out[m][n] = act(s(m, n) * (xs[m] * ws[n]) + bias[n]),
// s(m, n) = sum_k x[m][k] w[n][k] in 32-bit integers, act the identity or the tanh form of GELU.
//
// Output channels lie on the M side of the matrix instructions and tokens on the N side: weights
// come in whole multiples of 128 channels in practice, while the number of tokens is anything from
// one to a window, and the instruction's N side takes any multiple of 16 (32 for an SM pair).
// Integer sums are exact in any order, so how K is split changes no bit of the result.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>

#include "common.cuh"

namespace ss {

int encode_tmap_2d_u8(CUtensorMap *map, const void *base, uint64_t inner, uint64_t outer, uint64_t row_stride_bytes,
                      uint32_t box_inner, uint32_t box_outer);

namespace lin {

struct Params {
    const float *xs, *ws;
    const void *bias;
    int bias_dtype, gelu, out_dtype;
    int M, N, K;
    void *out;
    int64_t out_ld;
    int *status;
    int tn;      // tokens a tile
    int ncb;     // channel blocks
    int ntiles;  // channel blocks x token blocks (pairs)
    int vec;     // rows of out take 4-channel vector stores
};

__device__ __forceinline__ float load_any(const void *p, int dtype, int64_t i) {
    if (dtype == SS_F32) return static_cast<const float *>(p)[i];
    if (dtype == SS_F16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
template <int DT>
__device__ __forceinline__ void store_one(void *p, int64_t i, float v) {
    if (DT == SS_F32) static_cast<float *>(p)[i] = v;
    else if (DT == SS_F16) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

// tanh form of GELU, 0.5 v (1 + tanh(u)) = v / (1 + exp(-2u)), u = sqrt(2/pi) (v + 0.044715 v^3):
// no cancellation for negative v, and an exponential that overflows gives -0
__device__ __forceinline__ float gelu_tanh(float v) {
    const float u2 = 1.5957691216057308f * v * (1.f + 0.044715f * v * v);
    return v / (1.f + __expf(-u2));
}
__device__ __forceinline__ float finish(int acc, float s, float b, bool has_bias, bool gelu) {
    float v = __fmul_rn((float)acc, s);
    if (has_bias) v = __fadd_rn(v, b);
    return gelu ? gelu_tanh(v) : v;
}

// ---------------------------------------------------------------------------------------------
// clusters and SM pairs
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address of this CTA's shared-memory word at the same place in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// one CTA's half of a pair's load: into this CTA's shared memory, counted by a barrier of either CTA
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
// D[tmem] (+)= A[smem] * B[smem], kind::i8 (s8 inputs, s32 accumulate)
template <int CTAS>
__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
    if (CTAS == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
            : "memory");
}
// signals the barrier at this place in both CTAs of the pair once the MMAs issued so far are done
__device__ __forceinline__ void commit_both(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
        ::"r"(bar), "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void commit_pair_own(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// kind::i8 instruction descriptor: D s32, A and B signed 8-bit, both K-major
__host__ __device__ constexpr uint32_t idesc_i8(int M, int N) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ bool warp_all(bool ok) { return __all_sync(0xffffffffu, ok); }
// a wait that ignores the abort flag (only to drain work this CTA itself issued)
__device__ __forceinline__ bool drain_wait(uint32_t bar, uint32_t parity) {
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity))
        if (clock64() - t0 > kWaitLimitCycles) return false;
    return true;
}

constexpr int BK = 128;                          // codes a stage: one 128-byte swizzled row
constexpr uint32_t W_BYTES = 128 * BK;           // 128 channels of a stage
constexpr int STAGES = 6;

// ---------------------------------------------------------------------------------------------
// many tokens: an SM pair per tile of 256 channels x tn tokens
// ---------------------------------------------------------------------------------------------
// Persistent, one CTA per SM. Each CTA of a pair loads its 128 channels and half of the tile's
// tokens; the even CTA issues the pair's MMAs (M 256, N tn, K 32), whose 32-bit sums land in both
// CTAs' tensor memory, 128 channels each. Two accumulators of up to 256 columns let the eight
// epilogue warps of each CTA empty one tile while the next is summed.
namespace pair {

constexpr int EPI_WARPS = 8;
constexpr int THREADS = (EPI_WARPS + 2) * 32;
constexpr uint32_t X_BYTES = 128 * BK;           // half of 256 tokens
constexpr uint32_t STAGE_BYTES = W_BYTES + X_BYTES;
constexpr uint32_t OFF_BAR = STAGES * STAGE_BYTES;
enum Bar { FULL = 0, EMPTY = FULL + STAGES, ACC_FULL = EMPTY + STAGES, ACC_EMPTY = ACC_FULL + 2,
           DRAIN = ACC_EMPTY + 2, NBAR = DRAIN + 1 };
constexpr uint32_t OFF_MISC = OFF_BAR + NBAR * 8 + (NBAR % 2) * 8;   // [0] tmem, [1] abort
constexpr uint32_t OFF_XS = OFF_MISC + 16;
constexpr uint32_t SMEM_BYTES = OFF_XS + EPI_WARPS * 32 * 4 + 1024;         // + alignment slack

template <int DT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_u32(smem);
    auto bar = [&](int i) -> uint32_t { return sbase + OFF_BAR + 8u * (uint32_t)i; };
    volatile uint32_t *misc = reinterpret_cast<volatile uint32_t *>(smem + OFF_MISC);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + OFF_MISC + 4);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_rank();
    const int pair_id = blockIdx.x >> 1, npairs = gridDim.x >> 1;
    const int nk = (p.K + BK - 1) / BK;

    if (tid == 0) {
        for (int i = 0; i < NBAR; ++i)
            mbar_init(bar(i), (i == ACC_EMPTY || i == ACC_EMPTY + 1) ? 2 * EPI_WARPS : 1);
        fence_mbar_init();
        *abort_flag = 0;
        prefetch_tmap(&tm_w);
        prefetch_tmap(&tm_x);
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sbase + OFF_MISC),
                     "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        tc_fence_before();
    }
    __syncthreads();
    cluster_sync();   // both CTAs' barriers are initialised before either is signalled from the other
    tc_fence_after();
    const uint32_t tmem = misc[0];

    if (warp < EPI_WARPS) {
        // ---------------- epilogue: one channel per thread, every other 32 tokens ----------------
        const int wg = warp >> 2;
        const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const uint32_t acc_empty = in_cta(bar(ACC_EMPTY), 0);
        float *xs_s = reinterpret_cast<float *>(smem + OFF_XS) + warp * 32;   // the warp's 32 token scales
        bool ok = true;
        int it = 0;
        for (int tile = pair_id; tile < p.ntiles && ok; tile += npairs, ++it) {
            const int n = (tile % p.ncb) * 256 + (int)rank * 128 + 32 * (warp & 3) + lane;
            const int64_t m0 = (int64_t)(tile / p.ncb) * p.tn;
            const float wsv = n < p.N ? p.ws[n] : 0.f;
            const float bv = (p.bias && n < p.N) ? load_any(p.bias, p.bias_dtype, n) : 0.f;
            const int b = it & 1;
            ok = warp_all(mbar_wait(bar(ACC_FULL + b), (it >> 1) & 1, abort_flag));
            if (!ok) break;
            tc_fence_after();
            for (int c = wg; c < p.tn / 32; c += 2) {
                float v[32];
                tmem_ld32(lanes + 256 * b + 32 * c, v);
                const int64_t mc = m0 + 32 * c;
                __syncwarp();   // the chunk before has been read
                xs_s[lane] = mc + lane < p.M ? p.xs[mc + lane] : 0.f;
                __syncwarp();
                tmem_wait_ld();
                tmem_ld_fence32(v);
                const int rows = (int)min((int64_t)32, p.M - mc);
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    const float y = finish(__float_as_int(v[j]), __fmul_rn(xs_s[j], wsv), bv,
                                           p.bias != nullptr, p.gelu != 0);
                    if (j < rows && n < p.N) store_one<DT>(p.out, (mc + j) * p.out_ld + n, y);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc_empty + 8u * (uint32_t)b);
        }
        if (!ok) report(p.status, SS_DEV_TIMEOUT);
    } else if (warp == EPI_WARPS) {
        // ---------------- TMA producer (both CTAs) ----------------
        const uint32_t x_bytes = (uint32_t)(p.tn / 2) * BK;
        const uint32_t full = in_cta(bar(FULL), 0);
        int i = 0;   // stages issued
        bool ok = true;
        for (int tile = pair_id; tile < p.ntiles && ok; tile += npairs) {
            const int n0 = (tile % p.ncb) * 256 + (int)rank * 128;
            const int m0 = (tile / p.ncb) * p.tn + (int)rank * (p.tn / 2);
            for (int k = 0; k < nk; ++k, ++i) {
                const int st = i % STAGES;
                if (i >= STAGES) {
                    ok = warp_all(mbar_wait(bar(EMPTY + st), (i / STAGES - 1) & 1, abort_flag));
                    if (!ok) break;
                }
                if (elect_one()) {
                    const uint32_t dst = sbase + (uint32_t)st * STAGE_BYTES;
                    if (rank == 0) mbar_arrive_expect_tx(bar(FULL + st), 2 * (W_BYTES + x_bytes));
                    tma_load_2d_pair(dst, &tm_w, k * BK, n0, full + 8u * (uint32_t)st);
                    tma_load_2d_pair(dst + W_BYTES, &tm_x, k * BK, m0, full + 8u * (uint32_t)st);
                }
                __syncwarp();
            }
        }
        if (!ok) report(p.status, SS_DEV_TIMEOUT);
        if (!ok || *abort_flag) {
            // the loads still in flight land before the CTA's shared memory goes away: the even CTA sees
            // both CTAs' by its full barriers, the odd one only by the stages' release
            for (int s = i > STAGES ? i - STAGES : 0; s < i; ++s)
                drain_wait(bar((rank == 0 ? FULL : EMPTY) + s % STAGES), (s / STAGES) & 1);
        }
    } else if (rank == 0) {
        // ---------------- MMA issuer (the even CTA) ----------------
        const uint32_t idesc = idesc_i8(256, p.tn);
        int i = 0, it = 0;
        bool ok = true;
        for (int tile = pair_id; tile < p.ntiles && ok; tile += npairs, ++it) {
            const int b = it & 1;
            if (it >= 2) {
                ok = warp_all(mbar_wait(bar(ACC_EMPTY + b), ((it >> 1) - 1) & 1, abort_flag));
                if (!ok) break;
            }
            tc_fence_after();
            for (int k = 0; k < nk; ++k, ++i) {
                const int st = i % STAGES;
                ok = warp_all(mbar_wait(bar(FULL + st), (i / STAGES) & 1, abort_flag));
                if (!ok) break;
                tc_fence_after();
                const uint64_t da = smem_desc_sw128(sbase + (uint32_t)st * STAGE_BYTES, 16, 1024);
                const uint64_t db = smem_desc_sw128(sbase + (uint32_t)st * STAGE_BYTES + W_BYTES, 16, 1024);
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < BK / 32; ++kk)
                        mma_i8<2>(tmem + 256 * b, da + 2 * kk, db + 2 * kk, idesc, (k > 0 || kk > 0) ? 1u : 0u);
                    commit_both(bar(EMPTY + st));
                    if (k == nk - 1) commit_both(bar(ACC_FULL + b));
                }
                __syncwarp();
            }
        }
        if (!ok) report(p.status, SS_DEV_TIMEOUT);
        if (!ok || *abort_flag) {
            if (elect_one()) commit_pair_own(bar(DRAIN));   // arrives once every MMA issued so far is done
            __syncwarp();
            drain_wait(bar(DRAIN), 0);
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();   // neither CTA's memory goes away while the other may still signal or read it
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace pair

// ---------------------------------------------------------------------------------------------
// few tokens: a cluster per tile of 128 channels x tn tokens, K split over its CTAs
// ---------------------------------------------------------------------------------------------
// CTA r of a cluster of S sums its share of K in its tensor memory and lays the sums out in its
// shared memory as [token][channel]; after a cluster barrier it adds up every S-th part of the
// tokens over the S CTAs (distributed shared memory) and finishes those rows.
namespace split {

constexpr int THREADS = 192;   // warps 0-3: accumulator rows; 4: TMA; 5: MMA; all: the final rows
constexpr int MAX_TN = 128;
constexpr int MAX_S = 8;
enum Bar { FULL = 0, EMPTY = FULL + STAGES, ACC = EMPTY + STAGES, DRAIN = ACC + 1, NBAR = DRAIN + 1 };

__host__ __device__ constexpr uint32_t stage_bytes(int tn) { return W_BYTES + (uint32_t)tn * BK; }
__host__ __device__ constexpr uint32_t off_bar(int tn) { return STAGES * stage_bytes(tn); }
__host__ __device__ constexpr uint32_t smem_bytes(int tn) { return off_bar(tn) + NBAR * 8 + 32 + 1024; }
static_assert(STAGES * W_BYTES >= 128u * 128u * 4u, "the sums fit in the stages' memory");

template <int DT>
__global__ void __launch_bounds__(THREADS)
kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const Params p, int S) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_u32(smem);
    const uint32_t bars = sbase + off_bar(p.tn);
    auto bar = [&](int i) -> uint32_t { return bars + 8u * (uint32_t)i; };
    volatile uint32_t *misc = reinterpret_cast<volatile uint32_t *>(smem + off_bar(p.tn) + NBAR * 8);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + off_bar(p.tn) + NBAR * 8 + 4);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)(blockIdx.x % (unsigned)S), tile = (int)(blockIdx.x / (unsigned)S);
    const int n0 = (tile % p.ncb) * 128;
    const int m0 = (tile / p.ncb) * p.tn;
    const int nk = (p.K + BK - 1) / BK;
    const int k_lo = (int)((int64_t)rank * nk / S), k_hi = (int)((int64_t)(rank + 1) * nk / S);
    const uint32_t cols = p.tn <= 32 ? 32u : p.tn <= 64 ? 64u : 128u;

    if (tid == 0) {
        for (int i = 0; i < NBAR; ++i) mbar_init(bar(i), 1);
        fence_mbar_init();
        *abort_flag = 0;
        prefetch_tmap(&tm_w);
        prefetch_tmap(&tm_x);
    }
    if (warp == 0) {
        tmem_alloc(smem_u32(const_cast<uint32_t *>(misc)), cols);
        tmem_relinquish();
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = misc[0];
    int *sums = reinterpret_cast<int *>(smem);   // [tn][128], over the stages once they are consumed
    bool ok = true;

    if (warp == 4) {
        const uint32_t bytes = stage_bytes(p.tn);
        int i = 0;
        for (int k = k_lo; k < k_hi; ++k, ++i) {
            const int st = i % STAGES;
            if (i >= STAGES) {
                ok = warp_all(mbar_wait(bar(EMPTY + st), (i / STAGES - 1) & 1, abort_flag));
                if (!ok) break;
            }
            if (elect_one()) {
                const uint32_t dst = sbase + (uint32_t)st * bytes;
                mbar_arrive_expect_tx(bar(FULL + st), bytes);
                tma_load_2d(dst, &tm_w, k * BK, n0, bar(FULL + st));
                tma_load_2d(dst + W_BYTES, &tm_x, k * BK, m0, bar(FULL + st));
            }
            __syncwarp();
        }
        if (!ok) report(p.status, SS_DEV_TIMEOUT);
        if (!ok || *abort_flag)
            for (int s = i > STAGES ? i - STAGES : 0; s < i; ++s) drain_wait(bar(FULL + s % STAGES), (s / STAGES) & 1);
    } else if (warp == 5) {
        const uint32_t idesc = idesc_i8(128, p.tn), bytes = stage_bytes(p.tn);
        int i = 0;
        for (int k = k_lo; k < k_hi; ++k, ++i) {
            const int st = i % STAGES;
            ok = warp_all(mbar_wait(bar(FULL + st), (i / STAGES) & 1, abort_flag));
            if (!ok) break;
            tc_fence_after();
            const uint64_t da = smem_desc_sw128(sbase + (uint32_t)st * bytes, 16, 1024);
            const uint64_t db = smem_desc_sw128(sbase + (uint32_t)st * bytes + W_BYTES, 16, 1024);
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < BK / 32; ++kk)
                    mma_i8<1>(tmem, da + 2 * kk, db + 2 * kk, idesc, (i > 0 || kk > 0) ? 1u : 0u);
                tc_commit(bar(EMPTY + st));
                if (k == k_hi - 1) tc_commit(bar(ACC));
            }
            __syncwarp();
        }
        if (!ok) report(p.status, SS_DEV_TIMEOUT);
        if (!ok || *abort_flag) {
            if (elect_one()) tc_commit(bar(DRAIN));   // arrives once every MMA issued so far is done
            __syncwarp();
            drain_wait(bar(DRAIN), 0);
        }
    } else {
        ok = warp_all(mbar_wait(bar(ACC), 0, abort_flag));
        if (!ok) report(p.status, SS_DEV_TIMEOUT);
        if (ok) {
            tc_fence_after();
            const uint32_t lanes = tmem + ((uint32_t)(32 * warp) << 16);
            for (int c = 0; c < p.tn; c += 32) {   // tn may end 16 columns into the last 32
                float v[32];
                tmem_ld32(lanes + c, v);
                tmem_wait_ld();
                tmem_ld_fence32(v);
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (c + j < p.tn) sums[(c + j) * 128 + tid] = __float_as_int(v[j]);
            }
        }
    }
    tc_fence_before();
    if (S > 1) cluster_sync();
    else __syncthreads();
    // after a wait that ran out the sums are not whole, but the memory they are read from is there
    const int t_lo = rank * p.tn / S, t_hi = (rank + 1) * p.tn / S;
    for (int i = tid; i < (t_hi - t_lo) * 32; i += THREADS) {
        const int t = t_lo + i / 32, c = (i % 32) * 4;
        const int64_t m = (int64_t)m0 + t;
        if (m >= p.M) break;
        const uint32_t at = sbase + (uint32_t)(t * 128 + c) * 4u;
        int a[4] = {0, 0, 0, 0};
        for (int r = 0; r < S; ++r) {
            int b[4];
            if (S > 1)
                asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3]) : "r"(in_cta(at, (uint32_t)r)));
            else
                asm volatile("ld.shared.v4.s32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3]) : "r"(at));
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] += b[j];
        }
        const float xsv = p.xs[m];
        const int64_t at_out = m * p.out_ld + n0 + c;
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + c + j;
            y[j] = n < p.N ? finish(a[j], __fmul_rn(xsv, p.ws[n]), p.bias ? load_any(p.bias, p.bias_dtype, n) : 0.f,
                                    p.bias != nullptr, p.gelu != 0)
                           : 0.f;
        }
        if (p.vec && n0 + c + 3 < p.N) {
            if (DT == SS_F32) {
                *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at_out) = make_float4(y[0], y[1], y[2], y[3]);
            } else {
                union {
                    __nv_bfloat16 h[4];
                    __half f[4];
                    uint2 u;
                } o;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (DT == SS_F16) o.f[j] = __float2half_rn(y[j]);
                    else o.h[j] = __float2bfloat16_rn(y[j]);
                }
                *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + at_out) = o.u;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + c + j < p.N) store_one<DT>(p.out, at_out + j, y[j]);
        }
    }
    if (S > 1) cluster_sync();   // no CTA's sums go away while another reads them
    else __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, cols);
    }
}

}  // namespace split

static bool off(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }
static size_t type_bytes(int dtype) { return dtype == SS_F32 ? 4 : 2; }
static bool known(int dtype) { return dtype == SS_BF16 || dtype == SS_F32 || dtype == SS_F16; }

}  // namespace lin

static std::mutex g_lin_mutex;
static int g_lin_configured[SS_MAX_DEVICES];
static void *g_lin_ctx[SS_MAX_DEVICES];
static int g_lin_nsm[SS_MAX_DEVICES];

template <int DT>
static cudaError_t linear_i8_attributes() {
    cudaError_t e = cudaFuncSetAttribute(lin::pair::kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)lin::pair::SMEM_BYTES);
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(lin::split::kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)lin::split::smem_bytes(lin::split::MAX_TN));
}

int linear_i8_prepare(int device) {
    if (device < 0 || device >= SS_MAX_DEVICES) return SS_ERR_DEVICE;
    void *ctx = nullptr;
    int rc = current_context(&ctx);
    if (rc) return rc;
    std::lock_guard<std::mutex> lock(g_lin_mutex);
    if (g_lin_configured[device] && g_lin_ctx[device] == ctx) return 0;
    cudaError_t e = linear_i8_attributes<SS_BF16>();
    if (e == cudaSuccess) e = linear_i8_attributes<SS_F32>();
    if (e == cudaSuccess) e = linear_i8_attributes<SS_F16>();
    int nsm = 0;
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&nsm, cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess) return (int)e;
    g_lin_nsm[device] = nsm;
    g_lin_ctx[device] = ctx;
    g_lin_configured[device] = 1;
    return 0;
}

namespace lin {

struct Plan {
    bool pairs;
    int tn, S;
};

static Plan choose(int M, int N, int K, int nsm) {
    const int npairs = nsm / 2;
    const int64_t ncb2 = (N + 255) / 256, ncb = (N + 127) / 128;
    const int nk = (K + BK - 1) / BK;
    if (ncb2 * ((M + 255) / 256) * 2 >= npairs) {
        Plan best = {true, 256, 1};
        double cost = 1e30;
        for (int tn = 256; tn >= 96; tn -= 32) {
            const int64_t tiles = ncb2 * ((M + tn - 1) / tn);
            const double c = (double)((tiles + npairs - 1) / npairs) * (tn + 64);
            if (c < cost - 1e-9) cost = c, best.tn = tn;
        }
        return best;
    }
    Plan best = {false, 16, 1};
    best.tn = M >= split::MAX_TN ? split::MAX_TN : (M + 15) / 16 * 16;
    const int64_t tiles = ncb * ((M + best.tn - 1) / best.tn);
    while (best.S < split::MAX_S && tiles * best.S * 2 <= nsm && best.S * 2 <= nk) best.S *= 2;
    return best;
}

template <int DT>
static int launch(const Plan &plan, const int8_t *x, int64_t x_ld, const int8_t *w, int64_t w_ld, Params p, int nsm,
                  cudaStream_t st) {
    CUtensorMap tm_w, tm_x;
    p.tn = plan.tn;
    int rc = encode_tmap_2d_u8(&tm_w, w, (uint64_t)p.K, (uint64_t)p.N, (uint64_t)w_ld, BK, 128);
    if (!rc) rc = encode_tmap_2d_u8(&tm_x, x, (uint64_t)p.K, (uint64_t)p.M, (uint64_t)x_ld, BK,
                                    (uint32_t)(plan.pairs ? plan.tn / 2 : plan.tn));
    if (rc) return rc;
    const int64_t ntb = ((int64_t)p.M + plan.tn - 1) / plan.tn;
    if (plan.pairs) {
        p.ncb = (p.N + 255) / 256;
        const int64_t tiles = p.ncb * ntb;
        if (tiles > 0x7fffffff) return SS_ERR_SHAPE;
        p.ntiles = (int)tiles;
        const int npairs = (int)(tiles < nsm / 2 ? tiles : nsm / 2);
        pair::kernel<DT><<<2 * npairs, pair::THREADS, pair::SMEM_BYTES, st>>>(tm_w, tm_x, p);
        return (int)cudaGetLastError();
    }
    p.ncb = (p.N + 127) / 128;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.ncb * ntb * plan.S));
    cfg.blockDim = dim3(split::THREADS);
    cfg.dynamicSmemBytes = split::smem_bytes(plan.tn);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)plan.S;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, split::kernel<DT>, tm_w, tm_x, p, plan.S);
}

}  // namespace lin
}  // namespace ss

extern "C" int ss_linear_i8(const int8_t *x, int64_t x_ld, const float *xs, const int8_t *w, int64_t w_ld,
                            const float *ws, const void *bias, int bias_dtype, int gelu, int M, int N, int K,
                            void *out, int64_t out_ld, int out_dtype, int *status, void *stream) {
    using namespace ss;
    if (M < 0 || N <= 0 || K <= 0 || K > SS_LINEAR_I8_MAX_K || M > SS_LINEAR_I8_MAX_ROWS || N > SS_LINEAR_I8_MAX_ROWS || x_ld < K || w_ld < K || out_ld < N || (x_ld % 16) ||
        (w_ld % 16) || !lin::known(out_dtype) || (bias && !lin::known(bias_dtype)))
        return SS_ERR_SHAPE;
    if (M == 0) return 0;   // buffers without rows may have no address
    if (!x || !xs || !w || !ws || !out) return SS_ERR_POINTER;
    if (lin::off(x, 16) || lin::off(w, 16) || lin::off(xs, 4) || lin::off(ws, 4) || lin::off(status, 4) ||
        lin::off(out, lin::type_bytes(out_dtype)) || (bias && lin::off(bias, lin::type_bytes(bias_dtype))))
        return SS_ERR_POINTER;
    int device;
    const cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    const int rc = linear_i8_prepare(device);
    if (rc) return rc;
    const int nsm = g_lin_nsm[device];
    lin::Params p = {};
    p.xs = xs, p.ws = ws, p.bias = bias, p.bias_dtype = bias_dtype, p.gelu = gelu, p.out_dtype = out_dtype;
    p.M = M, p.N = N, p.K = K, p.out = out, p.out_ld = out_ld, p.status = status;
    p.vec = !lin::off(out, 4 * lin::type_bytes(out_dtype)) && out_ld % 4 == 0;
    const lin::Plan plan = lin::choose(M, N, K, nsm);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (out_dtype == SS_BF16) return lin::launch<SS_BF16>(plan, x, x_ld, w, w_ld, p, nsm, st);
    if (out_dtype == SS_F16) return lin::launch<SS_F16>(plan, x, x_ld, w, w_ld, p, nsm, st);
    return lin::launch<SS_F32>(plan, x, x_ld, w, w_ld, p, nsm, st);
}
