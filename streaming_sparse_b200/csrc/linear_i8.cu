// linear_i8.cu -- the 8-bit linear layer: out[m][n] = act(s(m, n) * (xs[m] * ws[n]) + bias[n]),
// s(m, n) = sum_k x[m][k] w[n][k] in 32-bit integers, act the identity or the tanh form of GELU.
//
// Output channels lie on the M side of the matrix instructions and tokens on the N side: weights
// come in whole multiples of 128 channels in practice, while the number of tokens is anything from
// one to a window, and the instruction's N side takes any multiple of 16 (32 for an SM pair).
// Integer sums are exact in any order, so how K is split changes no bit of the result.
//
// Three kernels: dot products for one to four tokens (weights' bytes), clusters that split K for few
// tokens (latency), SM pairs for many (L2 and the tensor pipe). Measured on B200 (CUDA-graph replay over buffers
// beyond L2, a fresh process each):
//   one token x 8960 x 1536, GELU          4.1 us, 3.3 TB/s of weights (2.9 us from L2)
//   77 x 1531 x 1549 to fp32               6.7 us
//   4680 x 4608 x 1536                    27.5 us, 2.41 POPS (34.5 us to fp32)
//   4680 x 8960 x 1536, GELU              54.7 us, 2.35 POPS (50.1 us without GELU)
//   4680 x 1536 x 1536                    12.7 us, 1.74 POPS
//   4680 x 1536 x 8960 to fp16            44.8 us, 2.88 POPS
//   32760 x 8960 x 1536, GELU       354 to 385 us, 2.3 to 2.5 POPS (the clocks fall under load)
// The library's 8-bit product of these sizes, which stops at the 32-bit sums: 29.8, 54.6, 48.7, 362 us (without the
// square one).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>

#include "common.cuh"
#include "launch.cuh"
#include "ring.cuh"

namespace ss {

int encode_tmap_2d_u8(CUtensorMap *map, const void *base, uint64_t inner, uint64_t outer, uint64_t row_stride_bytes,
                      uint32_t box_inner, uint32_t box_outer);
int encode_tmap_2d_b16_sw64(CUtensorMap *map, const void *base, uint64_t inner, uint64_t outer,
                            uint64_t row_stride_bytes, uint32_t box_inner, uint32_t box_outer);

namespace lin {

struct Params {
    const float *xs, *ws;
    const void *bias;
    int bias_dtype;
    int M, N, K;
    void *out;
    int64_t out_ld;
    int *status;
    int tn;      // tokens a tile
    int ncb;     // channel blocks
    int ntiles;  // channel blocks x token blocks (pairs)
    int vec;     // rows of out start at 16 bytes (pairs: TMA or 16-byte stores), 4 channels (split)
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

__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two finished values: act(float(acc) * s + b). The tanh form of GELU is computed as
// 0.5 v (1 + tanh(u)) = v / (1 + exp(-2u)), u = sqrt(2/pi) (v + 0.044715 v^3): no cancellation for
// negative v, and an exponential that overflows gives -0. The exponential is 2^(-2u log2(e)).
template <bool GELU>
__device__ __forceinline__ uint64_t finish(int acc0, int acc1, uint64_t s, uint64_t b) {
    const uint64_t v = f2_fma(f2((float)acc0, (float)acc1), s, b);
    if (!GELU) return v;
    constexpr float A = -2.302208198144325f;             // -2 sqrt(2/pi) log2(e)
    constexpr float B = A * 0.044715f;
    const uint64_t t = f2_mul(v, f2_fma(f2_mul(v, v), f2(B, B), f2(A, A)));
    return f2_mul(v, f2(rcp(1.f + ex2(f2_lo(t))), rcp(1.f + ex2(f2_hi(t)))));
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
// a box of this CTA's shared memory to the tensor at {x, y}, clipped to the tensor
__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, int x, int y, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(src)
                 : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// until all but the latest LEFT of this thread's bulk groups have read their shared memory
template <int LEFT>
__device__ __forceinline__ void bulk_read_wait() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LEFT) : "memory");
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
// 16 TMEM lanes x 32 columns as four 8-column fragments: v[4 i + 2 e + t] is lane 8 e + l / 4 (l this
// thread's lane in the warp), column 8 i + 2 (l % 4) + t
__device__ __forceinline__ void tmem_ld_16x256b_x4(uint32_t taddr, float *v) {
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// two values rounded to 16 bits, the first in the low half
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if (DT == SS_F16) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    return pack_bf16x2(lo, hi);
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

// ---------------------------------------------------------------------------------------------
// many tokens: an SM pair per tile of 256 channels x tn tokens
// ---------------------------------------------------------------------------------------------
// Persistent, one CTA per SM. Each CTA of a pair loads its 128 channels and half of the tile's
// tokens; the even CTA issues the pair's MMAs (M 256, N tn, K 32), whose 32-bit sums land in both
// CTAs' tensor memory, 128 channels each. Two accumulators of up to 256 columns let the sixteen
// epilogue warps of each CTA empty one tile while the next is summed.
//
// Why pairs: a CTA of its own needs 48 KB a step of 128 x 256 x 128 products, a pair's CTA 32 KB, and L2
// already delivers 17 TB/s at 256 x 256 (0.277 us a step, 0.27 at the tensor pipe's rate). What
// bounds it, by leaving parts out: 4680 x 8960 x 1536 takes 50.1 us, 41.1 without the stores of the 84 MB of
// outputs, 39.1 without the epilogue's arithmetic too, 38.5 without the epilogue: the stores, which share L2 with the
// loads. With GELU 54.7, 48.4, 39.0 and 38.5 us: its exponentials and reciprocals are not hidden either. 32-bit
// outputs of 4680 x 4608 x 1536, stored by the warps: 34.5 us, 23.6 without the stores, 20.7 without the epilogue. Eight epilogue warps were
// latency bound at two a scheduler (54.4 us, 64 with GELU against 56.3). 16-bit outputs leave as TMA boxes of
// 16 tokens x 32 channels; stored by the warps themselves they took 51.5 us (57 with GELU against 54.9).
namespace pair {

constexpr int EPI_WARPS = 16;
constexpr int THREADS = (EPI_WARPS + 2) * 32;
constexpr uint32_t RING_BYTES = 6 * 2 * W_BYTES;               // six stages of the largest tile
constexpr int MAX_STAGES = 10;
// per epilogue warp 2 KB: two halves of 16 tokens x 32 channels of 16 bits; or, for 32-bit outputs,
// 8 tokens x 32 channels and the token scales
constexpr uint32_t OFF_TURN = RING_BYTES;
constexpr uint32_t OFF_BAR = OFF_TURN + EPI_WARPS * 2048;
enum Bar { FULL = 0, EMPTY = FULL + MAX_STAGES, ACC_FULL = EMPTY + MAX_STAGES, ACC_EMPTY = ACC_FULL + 2,
           DRAIN = ACC_EMPTY + 2, NBAR = DRAIN + 1 };
constexpr uint32_t OFF_MISC = OFF_BAR + NBAR * 8 + (NBAR % 2) * 8;   // [0] tmem, [1] abort
constexpr uint32_t SMEM_BYTES = OFF_MISC + 16 + 1024;                // + alignment slack

__host__ __device__ constexpr uint32_t stage_bytes(int tn) { return W_BYTES + (uint32_t)(tn / 2) * BK; }
// a smaller tile's stages are smaller, and its loop waits for the loads' latency: more of them fit

template <int DT, bool GELU>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
       const __grid_constant__ CUtensorMap tm_out, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_u32(smem);
    constexpr int NCH = DT == SS_F32 ? 1 : 4;   // channels a thread
    auto bar = [&](int i) -> uint32_t { return sbase + OFF_BAR + 8u * (uint32_t)i; };
    volatile uint32_t *misc = reinterpret_cast<volatile uint32_t *>(smem + OFF_MISC);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + OFF_MISC + 4);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_rank();
    const int pair_id = blockIdx.x >> 1, npairs = gridDim.x >> 1;
    const int nk = (p.K + BK - 1) / BK;
    const uint32_t stage = stage_bytes(p.tn);
    const int nst = min((int)(RING_BYTES / stage), MAX_STAGES);

    if (tid == 0) {
        for (int i = 0; i < NBAR; ++i)
            mbar_init(bar(i), (i == ACC_EMPTY || i == ACC_EMPTY + 1) ? 2 * EPI_WARPS : 1);
        fence_mbar_init();
        *abort_flag = 0;
        prefetch_tmap(&tm_w);
        prefetch_tmap(&tm_x);
        if (DT != SS_F32 && p.vec) prefetch_tmap(&tm_out);
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
    let_next_start();
    wait_for_earlier();
    const uint32_t tmem = misc[0];

    if (warp < EPI_WARPS) {
        // ---------------- epilogue: 32 channels per warp, every fourth 32 tokens of the tile ----------------
        const int wg = warp >> 2;
        const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const uint32_t acc_empty = in_cta(bar(ACC_EMPTY), 0);
        const uint32_t turn = sbase + OFF_TURN + (uint32_t)warp * 2048;
        float *xs_w = reinterpret_cast<float *>(smem + OFF_TURN + warp * 2048 + 1024);   // 32-bit outputs: token scales
        bool ok = true;
        int it = 0;
        for (int tile = pair_id; tile < p.ntiles && ok; tile += npairs, ++it) {
            const int nw = (tile % p.ncb) * 256 + (int)rank * 128 + 32 * (warp & 3);   // the warp's channels
            const int64_t m0 = (int64_t)(tile / p.ncb) * p.tn;
            // rows that start at 16 bytes leave as TMA boxes, which clip to whole 16 bytes: not those that end inside one
            const bool boxes = p.vec && (p.N % 8 == 0 || nw + 32 <= p.N);
            // the channels this thread gets of an accumulator: lane (32-bit output), or lane / 4 + 8 i
            float wsv[NCH], bv[NCH];
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int n = nw + (DT == SS_F32 ? lane : (lane >> 2) + 8 * i);
                wsv[i] = n < p.N ? p.ws[n] : 0.f;
                bv[i] = (p.bias && n < p.N) ? load_any(p.bias, p.bias_dtype, n) : 0.f;
            }
            // the scales of the warp's tokens, 32-token chunks wg and wg + 4 of the tile: all of them in shared
            // memory, or this thread's tokens 8 i + 2 (lane % 4) + {0, 1} of each
            uint64_t xsv[2][4];
            if (DT == SS_F32) {
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int64_t m = m0 + 32 * (4 * i + wg) + lane;
                    if (32 * (4 * i + wg) < p.tn) xs_w[32 * i + lane] = m < p.M ? p.xs[m] : 0.f;
                }
                __syncwarp();
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int64_t m = m0 + 32 * (4 * (i >> 2) + wg) + 8 * (i & 3) + 2 * (lane & 3);
                    const bool in = 32 * (4 * (i >> 2) + wg) < p.tn;
                    xsv[i >> 2][i & 3] = f2(in && m < p.M ? p.xs[m] : 0.f, in && m + 1 < p.M ? p.xs[m + 1] : 0.f);
                }
            }
            const int b = it & 1;
            ok = warp_all(mbar_wait(bar(ACC_FULL + b), (it >> 1) & 1, abort_flag));
            if (!ok) break;
            tc_fence_after();
            const uint32_t acc = lanes + 256 * b;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int c = wg + 4 * u;
                if (c >= p.tn / 32) break;
                const int64_t mc = m0 + 32 * c;
                const int rows = (int)min((int64_t)32, p.M - mc);
                const float *xs_s = xs_w + 32 * u;
                float v[32];
                if (DT == SS_F32) {
                    tmem_ld32(acc + 32 * c, v);
                } else {   // 16 channels x 32 tokens twice, as 8 x 8 fragments
                    tmem_ld_16x256b_x4(acc + 32 * c, v);
                    tmem_ld_16x256b_x4(acc + 32 * c + (16u << 16), v + 16);
                }
                tmem_wait_ld();
                tmem_ld_fence32(v);
                if constexpr (DT == SS_F32) {
                    // thread = channel; 8 tokens at a time through shared memory, so that lane l stores
                    // channels 4 (l % 8) .. + 4 of a token
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        __syncwarp();   // the tokens before have left the warp's shared memory
#pragma unroll
                        for (int j = 0; j < 8; j += 2) {
                            const float2 x2 = *reinterpret_cast<const float2 *>(xs_s + 8 * h + j);
                            const uint64_t y = finish<GELU>(__float_as_int(v[8 * h + j]), __float_as_int(v[8 * h + j + 1]),
                                                            f2_mul(f2(x2.x, x2.y), f2(wsv[0], wsv[0])), f2(bv[0], bv[0]));
                            asm volatile("st.shared.f32 [%0], %1;" ::"r"(turn + 128u * j + 4u * lane), "f"(f2_lo(y)) : "memory");
                            asm volatile("st.shared.f32 [%0], %1;" ::"r"(turn + 128u * (j + 1) + 4u * lane), "f"(f2_hi(y)) : "memory");
                        }
                        __syncwarp();
                        const int nc = nw + 4 * (lane & 7);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int at = 4 * i + (lane >> 3), tok = 8 * h + at;
                            float u[4];
                            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                         : "=f"(u[0]), "=f"(u[1]), "=f"(u[2]), "=f"(u[3])
                                         : "r"(turn + 128u * at + 16u * (lane & 7)) : "memory");
                            if (tok < rows) {
                                float *dst = static_cast<float *>(p.out) + (mc + tok) * p.out_ld + nc;
                                if (p.vec && nc + 3 < p.N) {
                                    *reinterpret_cast<float4 *>(dst) = make_float4(u[0], u[1], u[2], u[3]);
                                } else {
#pragma unroll
                                    for (int j = 0; j < 4; ++j)
                                        if (nc + j < p.N) dst[j] = u[j];
                                }
                            }
                        }
                    }
                } else {
                    // v[16 h + 4 i + 2 e + t]: channel 16 h + 8 e + lane / 4, token 8 i + 2 (lane % 4) + t
                    const int nc = nw + 8 * (lane & 3);
#pragma unroll
                    for (int g = 0; g < 2; ++g) {   // 16 tokens at a time, in the two halves in turn
                        const uint32_t half = turn + 1024u * g;
                        if (lane == 0) bulk_read_wait<1>();   // the half's last store has read it
                        __syncwarp();
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int i = 2 * g + h;
                            uint32_t o[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int at = 16 * (e >> 1) + 4 * i + 2 * (e & 1);
                                const uint64_t y = finish<GELU>(__float_as_int(v[at]), __float_as_int(v[at + 1]),
                                                                f2_mul(xsv[u][i], f2(wsv[e % NCH], wsv[e % NCH])),
                                                                f2(bv[e % NCH], bv[e % NCH]));
                                o[e] = pack2<DT>(f2_lo(y), f2_hi(y));
                            }
                            // transposed into rows of 32 channels (64-byte swizzle): matrix e of the store is channels
                            // 8 e .. 8 e + 7 of tokens 8 i .. 8 i + 7, lane l gives the row of token 8 i + l % 8 of
                            // matrix l / 8
                            const int tok = 8 * h + (lane & 7);
                            const uint32_t to = half + (uint32_t)(tok * 64 + (((lane >> 3) ^ ((tok >> 1) & 3)) << 4));
                            asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};"
                                         ::"r"(to), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]) : "memory");
                        }
                        if (boxes) {
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                            __syncwarp();
                            if (lane == 0 && nw < p.N && 16 * g < rows) tma_store_2d(&tm_out, nw, (int)mc + 16 * g, half);
                        } else {   // lane l stores channels 8 (l % 4) .. + 8 of tokens l / 4 + 8 h one by one
                            __syncwarp();
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int at = 8 * h + (lane >> 2), tok = 16 * g + at;
                                const uint32_t from = half + (uint32_t)(at * 64 + (((lane & 3) ^ ((at >> 1) & 3)) << 4));
                                uint32_t w4[4];
                                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                             : "=r"(w4[0]), "=r"(w4[1]), "=r"(w4[2]), "=r"(w4[3]) : "r"(from) : "memory");
                                uint16_t *dst = static_cast<uint16_t *>(p.out) + (mc + tok) * p.out_ld + nc;
#pragma unroll
                                for (int j = 0; j < 8; ++j)
                                    if (tok < rows && nc + j < p.N) dst[j] = (uint16_t)(w4[j >> 1] >> (16 * (j & 1)));
                            }
                        }
                        if (lane == 0) bulk_commit();   // a group for every half, so that one left is the other half's
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc_empty + 8u * (uint32_t)b);
        }
        if (DT != SS_F32 && lane == 0) bulk_read_wait<0>();   // the shared memory stays until it has been read
        if (!ok) report(p.status, SS_DEV_LINEAR_TIMEOUT);
    } else if (warp == EPI_WARPS) {
        // ---------------- TMA producer (both CTAs) ----------------
        const uint32_t x_bytes = (uint32_t)(p.tn / 2) * BK;
        const uint32_t full = in_cta(bar(FULL), 0);
        Ring ring{nst};
        int issued = 0;
        bool ok = true;
        for (int tile = pair_id; tile < p.ntiles && ok; tile += npairs) {
            const int n0 = (tile % p.ncb) * 256 + (int)rank * 128;
            const int m0 = (tile / p.ncb) * p.tn + (int)rank * (p.tn / 2);
            for (int k = 0; k < nk; ++k) {
                // a fresh barrier counts as released: the first round does not wait
                ok = warp_all(mbar_wait(bar(EMPTY + ring.at), ring.parity ^ 1u, abort_flag));
                if (!ok) break;
                if (elect_one()) {
                    const uint32_t dst = sbase + (uint32_t)ring.at * stage;
                    if (rank == 0) mbar_arrive_expect_tx(bar(FULL + ring.at), 2 * (W_BYTES + x_bytes));
                    tma_load_2d_pair(dst, &tm_w, k * BK, n0, full + 8u * (uint32_t)ring.at);
                    tma_load_2d_pair(dst + W_BYTES, &tm_x, k * BK, m0, full + 8u * (uint32_t)ring.at);
                }
                __syncwarp();
                ring.next();
                issued = min(issued + 1, nst);
            }
        }
        // The even CTA's tensor core releases the stages of both CTAs by arrivals that nothing orders before the
        // last accumulator's: they reach this CTA's barriers before its shared memory goes away.
        if (ok)
            ok = ring.wait_for_each(issued, [&](int at, uint32_t parity) {
                return warp_all(mbar_wait(bar(EMPTY + at), parity, abort_flag));
            });
        if (!ok) report(p.status, SS_DEV_LINEAR_TIMEOUT);
        if (!ok || *abort_flag) {
            // the loads still in flight land before the CTA's shared memory goes away: the even CTA sees
            // both CTAs' by its full barriers, the odd one only by the stages' release
            ring.wait_for_each(issued, [&](int at, uint32_t parity) {
                drain_wait(bar((rank == 0 ? FULL : EMPTY) + at), parity);
                return true;
            });
        }
    } else if (rank == 0) {
        // ---------------- MMA issuer (the even CTA) ----------------
        const uint32_t idesc = idesc_i8(256, p.tn);
        const uint64_t dw = smem_desc_sw128(sbase, 16, 1024), dx = smem_desc_sw128(sbase + W_BYTES, 16, 1024);
        Ring ring{nst};
        int it = 0;
        bool ok = true;
        for (int tile = pair_id; tile < p.ntiles && ok; tile += npairs, ++it) {
            const int b = it & 1;
            ok = warp_all(mbar_wait(bar(ACC_EMPTY + b), ((it >> 1) & 1) ^ 1, abort_flag));
            if (!ok) break;
            tc_fence_after();
            for (int k = 0; k < nk; ++k) {
                ok = warp_all(mbar_wait(bar(FULL + ring.at), ring.parity, abort_flag));
                if (!ok) break;
                tc_fence_after();
                const uint64_t to = (uint64_t)((uint32_t)ring.at * stage >> 4);
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < BK / 32; ++kk)
                        mma_i8<2>(tmem + 256 * b, dw + to + 2 * kk, dx + to + 2 * kk, idesc, (k > 0 || kk > 0) ? 1u : 0u);
                    commit_both(bar(EMPTY + ring.at));
                    if (k == nk - 1) commit_both(bar(ACC_FULL + b));
                }
                __syncwarp();
                ring.next();
            }
        }
        if (!ok) report(p.status, SS_DEV_LINEAR_TIMEOUT);
        if (!ok || *abort_flag) {
            if (elect_one()) commit_pair_own(bar(DRAIN));   // arrives once every MMA issued so far is done
            __syncwarp();
            drain_wait(bar(DRAIN), 0);
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();   // neither CTA's memory goes away while the other's threads may still signal or read it
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
// tokens over the S CTAs (distributed shared memory) and finishes those rows. Bound by latency: about 4 us
// to start, load and finish, 0.2 us a step of K, so the split sets the time (16 x 1536 x 8960: 7.3 us over
// eight CTAs, 12.1 over two).
namespace split {

constexpr int THREADS = 192;   // warps 0-3: accumulator rows; 4: TMA; 5: MMA; all: the final rows
constexpr int MAX_TN = 128;
constexpr int MAX_S = 8;
constexpr int MAX_STAGES = 5;
enum Bar { FULL = 0, EMPTY = FULL + MAX_STAGES, ACC = EMPTY + MAX_STAGES, DRAIN = ACC + 1, NBAR = DRAIN + 1 };

__host__ __device__ constexpr uint32_t stage_bytes(int tn) { return W_BYTES + (uint32_t)tn * BK; }
// as many stages as leave room for two CTAs on an SM: a cluster of CTAs that each fill an SM leaves
// SMs idle where a GPC's SMs are no multiple of it
__host__ __device__ constexpr int stages(int tn) { return tn <= 32 ? 5 : tn <= 64 ? 4 : 3; }
__host__ __device__ constexpr uint32_t off_bar(int tn) { return stages(tn) * stage_bytes(tn); }
__host__ __device__ constexpr uint32_t smem_bytes(int tn) { return off_bar(tn) + NBAR * 8 + 32 + 1024; }
constexpr uint32_t MAX_SMEM = smem_bytes(32);
static_assert(MAX_SMEM >= smem_bytes(64) && MAX_SMEM >= smem_bytes(MAX_TN), "the largest of all tiles");
static_assert(off_bar(MAX_TN) >= MAX_TN * 512u && off_bar(64) >= 64 * 512u, "the sums fit in the stages' memory");

template <int DT, bool GELU, int S>
__global__ void __launch_bounds__(THREADS)
kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_u32(smem);
    const uint32_t bars = sbase + off_bar(p.tn);
    auto bar = [&](int i) -> uint32_t { return bars + 8u * (uint32_t)i; };
    volatile uint32_t *misc = reinterpret_cast<volatile uint32_t *>(smem + off_bar(p.tn) + NBAR * 8);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + off_bar(p.tn) + NBAR * 8 + 4);
    const int tid = threadIdx.x, warp = tid >> 5;
    const int rank = (int)(blockIdx.x % (unsigned)S), tile = (int)(blockIdx.x / (unsigned)S);
    const int n0 = (tile % p.ncb) * 128;
    const int m0 = (tile / p.ncb) * p.tn;
    const int nk = (p.K + BK - 1) / BK;
    const int k_lo = (int)((int64_t)rank * nk / S), k_hi = (int)((int64_t)(rank + 1) * nk / S);
    const int nst = stages(p.tn);
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
    let_next_start();
    wait_for_earlier();
    const uint32_t tmem = misc[0];
    int *sums = reinterpret_cast<int *>(smem);   // [tn][128], over the stages once they are consumed
    bool ok = true;

    if (warp == 4) {
        const uint32_t bytes = stage_bytes(p.tn);
        Ring ring{nst};
        int issued = 0;
        for (int k = k_lo; k < k_hi; ++k) {
            // a fresh barrier counts as released: the first round does not wait
            ok = warp_all(mbar_wait(bar(EMPTY + ring.at), ring.parity ^ 1u, abort_flag));
            if (!ok) break;
            if (elect_one()) {
                const uint32_t dst = sbase + (uint32_t)ring.at * bytes;
                mbar_arrive_expect_tx(bar(FULL + ring.at), bytes);
                tma_load_2d(dst, &tm_w, k * BK, n0, bar(FULL + ring.at));
                tma_load_2d(dst + W_BYTES, &tm_x, k * BK, m0, bar(FULL + ring.at));
            }
            __syncwarp();
            ring.next();
            issued = min(issued + 1, nst);
        }
        // the stages' last releases reach their barriers before the shared memory goes away
        if (ok)
            ok = ring.wait_for_each(issued, [&](int at, uint32_t parity) {
                return warp_all(mbar_wait(bar(EMPTY + at), parity, abort_flag));
            });
        if (!ok) report(p.status, SS_DEV_LINEAR_TIMEOUT);
        if (!ok || *abort_flag)   // the loads in flight land before the shared memory goes away
            ring.wait_for_each(issued, [&](int at, uint32_t parity) {
                drain_wait(bar(FULL + at), parity);
                return true;
            });
    } else if (warp == 5) {
        const uint32_t idesc = idesc_i8(128, p.tn), bytes = stage_bytes(p.tn);
        const uint64_t dw = smem_desc_sw128(sbase, 16, 1024), dx = smem_desc_sw128(sbase + W_BYTES, 16, 1024);
        Ring ring{nst};
        for (int k = k_lo; k < k_hi; ++k) {
            ok = warp_all(mbar_wait(bar(FULL + ring.at), ring.parity, abort_flag));
            if (!ok) break;
            tc_fence_after();
            const uint64_t to = (uint64_t)((uint32_t)ring.at * bytes >> 4);
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < BK / 32; ++kk)
                    mma_i8<1>(tmem, dw + to + 2 * kk, dx + to + 2 * kk, idesc, (k > k_lo || kk > 0) ? 1u : 0u);
                tc_commit(bar(EMPTY + ring.at));
                if (k == k_hi - 1) tc_commit(bar(ACC));
            }
            __syncwarp();
            ring.next();
        }
        if (!ok) report(p.status, SS_DEV_LINEAR_TIMEOUT);
        if (!ok || *abort_flag) {
            if (elect_one()) tc_commit(bar(DRAIN));   // arrives once every MMA issued so far is done
            __syncwarp();
            drain_wait(bar(DRAIN), 0);
        }
    } else {
        ok = warp_all(mbar_wait(bar(ACC), 0, abort_flag));
        if (!ok) report(p.status, SS_DEV_LINEAR_TIMEOUT);
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
    // each thread keeps its four channels: 32 threads a token
#pragma unroll 2
    for (int i = tid; i < (t_hi - t_lo) * 32; i += THREADS) {
        const int t = t_lo + i / 32, c = (i % 32) * 4;
        const int64_t m = (int64_t)m0 + t;
        if (m >= p.M) break;
        const uint32_t at = sbase + (uint32_t)(t * 128 + c) * 4u;
        int b[S][4], a[4] = {0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < S; ++r) {
            if (S > 1)
                asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(b[r][0]), "=r"(b[r][1]), "=r"(b[r][2]), "=r"(b[r][3])
                             : "r"(in_cta(at, (uint32_t)r)));
            else
                asm volatile("ld.shared.v4.s32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(b[r][0]), "=r"(b[r][1]), "=r"(b[r][2]), "=r"(b[r][3]) : "r"(at));
        }
#pragma unroll
        for (int r = 0; r < S; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] += b[r][j];
        const float xsv = p.xs[m];
        const int64_t at_out = m * p.out_ld + n0 + c;
        float wsv[4], bv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + c + j;
            wsv[j] = n < p.N ? p.ws[n] : 0.f;
            bv[j] = (p.bias && n < p.N) ? load_any(p.bias, p.bias_dtype, n) : 0.f;
        }
        const uint64_t y01 = finish<GELU>(a[0], a[1], f2_mul(f2(xsv, xsv), f2(wsv[0], wsv[1])), f2(bv[0], bv[1]));
        const uint64_t y23 = finish<GELU>(a[2], a[3], f2_mul(f2(xsv, xsv), f2(wsv[2], wsv[3])), f2(bv[2], bv[3]));
        const float y[4] = {f2_lo(y01), f2_hi(y01), f2_lo(y23), f2_hi(y23)};
        if (p.vec && n0 + c + 3 < p.N) {
            if (DT == SS_F32) {
                *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at_out) = make_float4(y[0], y[1], y[2], y[3]);
            } else {
                *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + at_out) =
                    make_uint2(pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3]));
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

// ---------------------------------------------------------------------------------------------
// one to four tokens: dot products
// ---------------------------------------------------------------------------------------------
// The weights are read once, straight to registers, 16 bytes a lane; WPC warps of a block share a
// group of CH channels, each taking every WPC-th 512 bytes of their rows. Lanes' sums meet by
// redux, warps' through shared memory. Bytes past K of a row's last 16 count as 0 through x. Bound by
// the weights' bytes and a launch: 8960 x 1536 weights 4.1 us (floor 2.1), 4.7 with four tokens, where five
// take 6.6 through the tensor cores; a form for eight tokens took 9.2, so four is the limit.
namespace dot {

constexpr int WARPS = 8;

template <int DT, bool GELU, int MT, int CH, int WPC>
__global__ void __launch_bounds__(WARPS * 32)
kernel(const int8_t *x, int64_t x_ld, const int8_t *w, int64_t w_ld, const Params p) {
    __shared__ int red[WARPS][CH * MT];
    let_next_start();
    wait_for_earlier();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % WPC;
    const int n0 = (blockIdx.x * (WARPS / WPC) + warp / WPC) * CH;
    const int chunks = (p.K + 15) / 16;
    const uint4 *wr[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) wr[c] = reinterpret_cast<const uint4 *>(w + (int64_t)min(n0 + c, p.N - 1) * w_ld);
    int acc[CH][MT] = {};
#pragma unroll 4
    for (int k = part * 32 + lane; k < chunks; k += WPC * 32) {
        uint4 a[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c)
            // not .nc: this kernel may have started before the one that wrote its inputs ended
            asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(a[c].x), "=r"(a[c].y), "=r"(a[c].z), "=r"(a[c].w) : "l"(wr[c] + k));
        const int left = p.K - 16 * k;   // codes of this chunk that are the row's
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            uint4 b = reinterpret_cast<const uint4 *>(x + (int64_t)min(m, p.M - 1) * x_ld)[k];
            if (left < 16) {
                uint32_t *e = &b.x;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    e[j] &= left >= 4 * j + 4 ? ~0u : left <= 4 * j ? 0u : (1u << (8 * (left - 4 * j))) - 1u;
            }
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                acc[c][m] = __dp4a((int)a[c].x, (int)b.x, acc[c][m]);
                acc[c][m] = __dp4a((int)a[c].y, (int)b.y, acc[c][m]);
                acc[c][m] = __dp4a((int)a[c].z, (int)b.z, acc[c][m]);
                acc[c][m] = __dp4a((int)a[c].w, (int)b.w, acc[c][m]);
            }
        }
    }
    int mine = 0;   // lane c MT + m keeps the sum of channel c and token m
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int t = __reduce_add_sync(0xffffffffu, acc[c][m]);
            if (lane == c * MT + m) mine = t;
        }
    if (WPC > 1) {
        if (lane < CH * MT) red[warp][lane] = mine;
        __syncthreads();
        if (part != 0) return;
        if (lane < CH * MT)
#pragma unroll
            for (int i = 1; i < WPC; ++i) mine += red[warp + i][lane];
    }
    const int n = n0 + lane / MT, m = lane % MT;
    if (lane < CH * MT && n < p.N && m < p.M) {
        const float s = __fmul_rn(p.xs[m], p.ws[n]), b = p.bias ? load_any(p.bias, p.bias_dtype, n) : 0.f;
        store_one<DT>(p.out, m * p.out_ld + n, f2_lo(finish<GELU>(mine, 0, f2(s, 0.f), f2(b, 0.f))));
    }
}

template <int DT, bool GELU, int MT, int CH>
static int launch(const int8_t *x, int64_t x_ld, const int8_t *w, int64_t w_ld, const Params &p, int nsm,
                  cudaStream_t st) {
    // enough warps for 16 an SM, as long as each has 512 bytes of a row to read
    const int64_t groups = (p.N + CH - 1) / CH;
    const int steps = (p.K + 511) / 512;
    int wpc = 1;
    while (wpc < WARPS && groups * wpc < 16 * (int64_t)nsm && wpc * 2 <= steps) wpc *= 2;
    const unsigned blocks = (unsigned)((groups * wpc + WARPS - 1) / WARPS);
    if (wpc == 1) return (int)launch_after(kernel<DT, GELU, MT, CH, 1>, blocks, WARPS * 32, 0, st, 1, x, x_ld, w, w_ld, p);
    if (wpc == 2) return (int)launch_after(kernel<DT, GELU, MT, CH, 2>, blocks, WARPS * 32, 0, st, 1, x, x_ld, w, w_ld, p);
    if (wpc == 4) return (int)launch_after(kernel<DT, GELU, MT, CH, 4>, blocks, WARPS * 32, 0, st, 1, x, x_ld, w, w_ld, p);
    return (int)launch_after(kernel<DT, GELU, MT, CH, 8>, blocks, WARPS * 32, 0, st, 1, x, x_ld, w, w_ld, p);
}

}  // namespace dot

static bool off(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }
static size_t type_bytes(int dtype) { return dtype == SS_F32 ? 4 : 2; }
static bool known(int dtype) { return dtype == SS_BF16 || dtype == SS_F32 || dtype == SS_F16; }

}  // namespace lin

static std::mutex g_lin_mutex;
static int g_lin_configured[SS_MAX_DEVICES];
static void *g_lin_ctx[SS_MAX_DEVICES];
static int g_lin_nsm[SS_MAX_DEVICES];

template <typename F>
static cudaError_t linear_i8_split_attributes(F kernel) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)lin::split::MAX_SMEM);
}
template <int DT, bool GELU>
static cudaError_t linear_i8_attributes() {
    cudaError_t e = cudaFuncSetAttribute(lin::pair::kernel<DT, GELU>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)lin::pair::SMEM_BYTES);
    if (e == cudaSuccess) e = linear_i8_split_attributes(lin::split::kernel<DT, GELU, 1>);
    if (e == cudaSuccess) e = linear_i8_split_attributes(lin::split::kernel<DT, GELU, 2>);
    if (e == cudaSuccess) e = linear_i8_split_attributes(lin::split::kernel<DT, GELU, 4>);
    if (e == cudaSuccess) e = linear_i8_split_attributes(lin::split::kernel<DT, GELU, 8>);
    return e;
}

int linear_i8_prepare(int device) {
    if (device < 0 || device >= SS_MAX_DEVICES) return SS_ERR_DEVICE;
    void *ctx = nullptr;
    int rc = current_context(&ctx);
    if (rc) return rc;
    std::lock_guard<std::mutex> lock(g_lin_mutex);
    if (g_lin_configured[device] && g_lin_ctx[device] == ctx) return 0;
    cudaError_t e = linear_i8_attributes<SS_BF16, false>();
    if (e == cudaSuccess) e = linear_i8_attributes<SS_BF16, true>();
    if (e == cudaSuccess) e = linear_i8_attributes<SS_F32, false>();
    if (e == cudaSuccess) e = linear_i8_attributes<SS_F32, true>();
    if (e == cudaSuccess) e = linear_i8_attributes<SS_F16, false>();
    if (e == cudaSuccess) e = linear_i8_attributes<SS_F16, true>();
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

// Which kernel and tile, by a model of the time in us: a launch, then for each round of tiles the steps
// over K and the tile's output. The constants are a fit to measured times (both kernels, every tile and
// split, 5 to 4680 tokens x five weights of 1536 x 1536 to 8960 x 1536 and 1536 x 8960; bf16 without GELU, before
// the kernels started early and stored boxes). As they are now the plan picked is 3 % off the fastest of these on
// average and 18 % at worst (4096 x 4096 weights, 96 tokens), with fp32 outputs or GELU 3 and 13 %. What it weighs (us):
// 16 tokens x 1536 x 8960 weights, 7.3 split over clusters of 8 against 16.2 in pairs, whose steps follow one another;
// 128 tokens x 4608 x 1536, 6.5 in pairs against 7.6 in single CTAs, whose weights are read by twice the CTAs.
static Plan choose(int M, int N, int K, int nsm) {
    const int npairs = nsm / 2;
    const int64_t ncb2 = (N + 255) / 256, ncb = (N + 127) / 128;
    const int nk = (K + BK - 1) / BK;
    Plan best = {true, 256, 1};
    double least = 1e30;
    for (int tn = 32; tn <= 256; tn += 32) {
        if (tn > 32 && tn - 32 >= M) break;
        const int64_t rounds = (ncb2 * ((M + tn - 1) / tn) + npairs - 1) / npairs;
        // a step takes 0.18 us to hand on (0.2 with stores of earlier tiles under way); from 192 tokens its
        // MMAs take longer
        const double step = tn <= 160 ? (rounds > 1 ? 0.2 : 0.18) : 0.00108 * tn;
        const double t = 4.5 + 0.01 * tn + (double)rounds * (nk * step + 0.2 + 0.004 * tn);
        if (t < least) least = t, best = {true, tn, 1};
    }
    for (int tn = 16; tn <= split::MAX_TN; tn += 16) {
        if (tn > 16 && tn - 16 >= M) break;
        const int64_t tiles = ncb * ((M + tn - 1) / tn);
        if (tiles > 2 * nsm) continue;
        for (int S = 1; S <= split::MAX_S && S <= nk; S *= 2) {
            const int64_t rounds = (tiles * S + nsm - 1) / nsm;
            const double step = 0.2 + 0.0012 * tn;
            const double t = 4.1 + (double)rounds * (step * ((nk + S - 1) / S) + 0.04 * tn) + 1.5 * (double)(rounds - 1);
            if (t < least) least = t, best = {false, tn, S};
        }
    }
    return best;
}

template <int DT, bool GELU>
static int launch(const Plan &plan, const int8_t *x, int64_t x_ld, const int8_t *w, int64_t w_ld, Params p, int nsm,
                  cudaStream_t st) {
    if (p.M == 1) return dot::launch<DT, GELU, 1, 2>(x, x_ld, w, w_ld, p, nsm, st);
    if (p.M == 2) return dot::launch<DT, GELU, 2, 2>(x, x_ld, w, w_ld, p, nsm, st);
    if (p.M <= 4) return dot::launch<DT, GELU, 4, 2>(x, x_ld, w, w_ld, p, nsm, st);
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
        CUtensorMap tm_out = {};
        if (DT != SS_F32 && p.vec) {
            rc = encode_tmap_2d_b16_sw64(&tm_out, p.out, (uint64_t)p.N, (uint64_t)p.M, (uint64_t)p.out_ld * 2, 32, 16);
            if (rc) return rc;
        }
        return (int)launch_after(pair::kernel<DT, GELU>, 2u * (unsigned)npairs, pair::THREADS, pair::SMEM_BYTES, st, 1, tm_w,
                                 tm_x, tm_out, p);
    }
    p.ncb = (p.N + 127) / 128;
    const unsigned blocks = (unsigned)(p.ncb * ntb * plan.S);
    const size_t smem = split::smem_bytes(plan.tn);
    auto go = [&](auto kernel) {
        return (int)launch_after(kernel, blocks, split::THREADS, smem, st, (unsigned)plan.S, tm_w, tm_x, p);
    };
    if (plan.S == 1) return go(split::kernel<DT, GELU, 1>);
    if (plan.S == 2) return go(split::kernel<DT, GELU, 2>);
    if (plan.S == 4) return go(split::kernel<DT, GELU, 4>);
    return go(split::kernel<DT, GELU, 8>);
}

}  // namespace lin
}  // namespace ss

extern "C" int ss_linear_i8(const int8_t *x, int64_t x_ld, const float *xs, const int8_t *w, int64_t w_ld,
                            const float *ws, const void *bias, int bias_dtype, int gelu, int M, int N, int K,
                            void *out, int64_t out_ld, int out_dtype, int *status, void *stream) {
    using namespace ss;
    if (M < 0 || N <= 0 || K <= 0 || K > SS_LINEAR_I8_MAX_K || M > SS_LINEAR_I8_MAX_ROWS ||
        N > SS_LINEAR_I8_MAX_ROWS || x_ld < K || w_ld < K || out_ld < N || (x_ld % 16) || (w_ld % 16) ||
        !lin::known(out_dtype) || (bias && !lin::known(bias_dtype)))
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
    p.xs = xs, p.ws = ws, p.bias = bias, p.bias_dtype = bias_dtype;
    p.M = M, p.N = N, p.K = K, p.out = out, p.out_ld = out_ld, p.status = status;
    const lin::Plan plan = lin::choose(M, N, K, nsm);
    const size_t store = plan.pairs ? 16 : 4 * lin::type_bytes(out_dtype);   // bytes of a vector store
    p.vec = !lin::off(out, store) && (size_t)out_ld * lin::type_bytes(out_dtype) % store == 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto go = [&](auto f) { return f(plan, x, x_ld, w, w_ld, p, nsm, st); };
    if (out_dtype == SS_BF16) return go(gelu ? lin::launch<SS_BF16, true> : lin::launch<SS_BF16, false>);
    if (out_dtype == SS_F16) return go(gelu ? lin::launch<SS_F16, true> : lin::launch<SS_F16, false>);
    return go(gelu ? lin::launch<SS_F32, true> : lin::launch<SS_F32, false>);
}
