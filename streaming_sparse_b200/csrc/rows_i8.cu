// rows_i8.cu -- 8-bit rows with one scale each: the row quantiser and the norms that end in it.
//
//   ss_quant_rows   s = max(max|x| / 127, 1e-30);  q = rint(x * (1 / s))
//   ss_rms_norm_i8  v = x + residual;  t = v * w;  u = max(max|t| / 127, 1e-30);
//                   q = rint(t * (1 / u));  s = u * rsqrt(mean(v^2) + eps)
//                   (the row's rsqrt is a common factor of its values, so it goes into the scale
//                   and the codes need no statistic but the maximum: one pass gives both)
//   ss_adaln_i8     v = x + y * gate[f];  z = (v - mean) * rsqrt(var + eps);
//                   o = z * (1 + scale[f]) + shift[f]  or  z * w + b;
//                   s = max(max|o| / 127, 1e-30);  q = rint(o * (1 / s))
// The sum v is also stored, rounded once to the rows' type; the norm reads it unrounded. All
// statistics are fp32. A row that holds an infinity or a NaN where its codes are made, or whose squares'
// sum overflows fp32, gets codes 0 and scale NaN, so that the products it enters are NaN and no other row's are.
//
// Bound: bytes. Each input is read once and each output written once; a row stays in registers between
// its statistics and its codes. Measured on B200 (bf16; the inputs', outputs' and codes' bytes over the time of a
// launch in a CUDA graph of twenty or more over buffers beyond L2, so that but for the last ones' tail the writes
// are in the time too). In the same way a copy of 32760 x 1536 reaches 6.3 TB/s, an addition (two reads a write)
// 6.8, of 131040 x 1536 6.6 and 7.0: reads go faster than writes, so what a plain copy reaches is no limit here.
//   quantiser                        4680 x 8960 20.6 us (6.1 TB/s), 20000 x 5120 44.5 us (6.9)
//   RMSNorm, residual's addition     32760 x 1536 53.7 us (6.6), 131040 x 1536 204 us (6.9), 4680 x 1536 10.6 us (4.7: two
//                                    waves of blocks; 6.2 us from L2)
//   AdaLN, gated addition            32760 x 1536 61 us (5.8), 4680 x 1536 13.7 us (9.5 us from L2); without the gate
//                                    11.9, affine with it 15.6, without an addition 8.1 us (5.9 us from L2)
// AdaLN reads three fp32 vectors a row through L1, 18 KB beside the row's own 10.8 KB, and reduces three times: L1's
// passes and the reductions' chains bound it, not HBM.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "launch.cuh"

namespace ss {
namespace rows {

constexpr float TINY = 1e-30f;   // the smallest scale: a row of zeros keeps a finite reciprocal

enum Mode { QUANT, RMS, MOD, AFFINE };   // MOD, AFFINE: the two forms of the LayerNorm

struct Args {
    const void *x;
    int64_t x_ld;
    const void *res;        // residual / y (null: none)
    int64_t res_ld;
    const float *gate;      // LN: per-frame gate rows (null: 1)
    int64_t gate_ld;
    const void *weight;     // RMS, affine LN
    const void *bias;       // affine LN
    const float *shift;     // modulated LN
    const float *scale;
    int64_t mod_ld;
    void *sum;
    int64_t sum_ld;
    int8_t *out;
    int64_t out_ld;
    float *scales;
    int n, d, frame_tokens;
    float eps, inv_d;       // inv_d = 1 / d
    int out_words;          // the codes of a chunk leave as one aligned word
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f(float v, float &o) { o = v; }
__device__ __forceinline__ void from_f(float v, __nv_bfloat16 &o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f(float v, __half &o) { o = __float2half_rn(v); }

// Magnitudes are compared as floats that keep a NaN, and between threads by their bits, whose order as
// unsigned integers is the finite numbers, infinity, the NaNs.
// the larger magnitude; a NaN stays one
__device__ __forceinline__ float max_abs(float m, float x) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
    return r;
}

// two sums that no product before them is fused into
__device__ __forceinline__ uint64_t add_both(uint64_t a, uint64_t b) {
    return f2(__fadd_rn(f2_lo(a), f2_lo(b)), __fadd_rn(f2_hi(a), f2_hi(b)));
}

struct Scale {
    float s, inv;
    uint32_t keep;   // all ones; 0 in a row whose codes are 0
};
// the scale of a row from the largest magnitude's bits; codes rint(x * inv) are within +-127
__device__ __forceinline__ Scale row_scale(uint32_t m) {
    if (m >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.f, 0u};
    const float s = fmaxf(__fdiv_rn(__uint_as_float(m), 127.f), TINY);
    return {s, __frcp_rn(s), ~0u};
}
// 1 / sqrt(mean + eps) of a row's squares. Where their sum overflowed it would be 0 and the row's codes would
// look like another row's: NaN, so that the row counts as not finite.
__device__ __forceinline__ float inv_root(float mean, float eps) {
    const float r = rsqrtf(__fadd_rn(mean, eps));
    return r > 0.f ? r : __uint_as_float(0x7fc00000u);
}
// the code of x is the low byte: adding 1.5 * 2^23 rounds |x| < 2^22 to the nearest integer, ties to even
constexpr float ROUND = 12582912.f;
__device__ __forceinline__ uint32_t code(float x, Scale s) {
    return __float_as_uint(__fadd_rn(__fmul_rn(x, s.inv), ROUND)) & s.keep;
}

// The block's reductions: warps by shuffles, then one word a warp through shared memory, with one
// barrier each (consecutive reductions use the two halves of `red` in turn). Every thread adds the
// warps' words in the same order.
template <bool WARP>
struct Reduce {
    float2 (*red)[32];
    int turn = 0;
    __device__ __forceinline__ float2 operator()(float s, uint32_t m) {   // (sum of s, max of m's bits)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        m = __reduce_max_sync(0xffffffffu, m);
        if (WARP || blockDim.x == 32) return make_float2(s, __uint_as_float(m));
        const int nw = blockDim.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) red[turn][threadIdx.x >> 5] = make_float2(s, __uint_as_float(m));
        __syncthreads();
        if (nw <= 8) {
            float2 a = red[turn][0];
            uint32_t top = __float_as_uint(a.y);
            for (int i = 1; i < nw; ++i) {
                const float2 b = red[turn][i];
                a.x += b.x;
                top = max(top, __float_as_uint(b.y));
            }
            a.y = __uint_as_float(top);
            turn ^= 1;
            return a;
        }
        const float2 a = lane < nw ? red[turn][lane] : make_float2(0.f, 0.f);
        s = a.x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        turn ^= 1;
        return make_float2(s, __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(a.y))));
    }
    __device__ __forceinline__ float sum(float s) { return (*this)(s, 0u).x; }
    __device__ __forceinline__ uint32_t max_bits(uint32_t m) { return __float_as_uint((*this)(0.f, m).y); }
};

// Consecutive values a thread takes at a time. The LayerNorms take four: their fp32 vectors then come as
// 16 bytes a lane without gaps. With eight (16 bytes of the 16-bit row) each lane's 32 bytes of a vector
// come as two loads of every other 16 bytes, twice the passes through L1, which bounded the kernel
// (32760 x 1536 AdaLN of bf16 45.6 us).
template <typename T, int MODE, bool AL>
__host__ __device__ constexpr int chunk_values() {
    return AL && MODE < MOD ? 16 / (int)sizeof(T) : 4;
}

// VEC values of a row of d from c on, as loaded: 8 or 16 bytes at once (AL: the chunk lies in the row), or
// one by one, with zeros past the row's end. FULL: no store lies past it.
template <typename T, int VEC, bool AL, bool FULL>
struct Chunk {
    static constexpr int BYTES = VEC * (int)sizeof(T), WORDS = BYTES <= 16 ? 1 : BYTES / 16;
    using Word = typename std::conditional<BYTES == 8, uint2, uint4>::type;
    union {
        Word u[WORDS];
        T e[VEC];
    };
    __device__ __forceinline__ Chunk() {}
    __device__ __forceinline__ void load(const T *src, int c, int d) {
        if constexpr (AL) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i)
                u[i] = reinterpret_cast<const Word *>(src + c)[i];
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                T z;
                from_f(0.f, z);
                e[j] = c + j < d ? src[c + j] : z;
            }
        }
    }
    __device__ __forceinline__ void store(T *dst, int c, int d) const {
        if constexpr (AL) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i)
                if (FULL || c < d) reinterpret_cast<Word *>(dst + c)[i] = u[i];
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (c + j < d) dst[c + j] = e[j];
        }
    }
    // values 2 j and 2 j + 1
    __device__ __forceinline__ uint64_t operator[](int j) const { return f2(to_f(e[2 * j]), to_f(e[2 * j + 1])); }
    __device__ __forceinline__ void set(int j, uint64_t v) {
        from_f(f2_lo(v), e[2 * j]);
        from_f(f2_hi(v), e[2 * j + 1]);
    }
};

template <int VEC, bool FULL>
__device__ __forceinline__ void store_codes(int8_t *out, int c, int d, int words, const uint64_t (&v)[VEC / 2], Scale s) {
    uint32_t k[VEC];
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) {
        const uint64_t y = f2_mul(v[j], f2(s.inv, s.inv));
        k[2 * j] = __float_as_uint(__fadd_rn(f2_lo(y), ROUND));
        k[2 * j + 1] = __float_as_uint(__fadd_rn(f2_hi(y), ROUND));
    }
    uint32_t o[VEC / 4];
#pragma unroll
    for (int j = 0; j < VEC / 4; ++j)
        o[j] = s.keep & __byte_perm(__byte_perm(k[4 * j], k[4 * j + 1], 0x0040),
                                    __byte_perm(k[4 * j + 2], k[4 * j + 3], 0x0040), 0x5410);
    if (words && (FULL || c + VEC <= d)) {
        if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(out + c) = make_uint2(o[0], o[1]);
        else *reinterpret_cast<uint32_t *>(out + c) = o[0];
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (FULL || c + j < d) out[c + j] = (int8_t)(o[j / 4] >> (8 * (j % 4)));
    }
}

__device__ __forceinline__ void prefetch_l1(const float *p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }

// The row in registers, NE values a thread: one read of each input, one write of each output. WARP: a
// warp per row (four rows a block), reductions by shuffles alone; else a block per row, as many threads
// as its chunks need. Thread t takes chunks t, t + threads, ... of VEC consecutive values, each a single
// load where base and strides allow (AL), else value by value in chunks of four, so that the codes still
// leave as whole words. All of x and the residual is asked for before the first value is used or the sum
// is stored: the sum may lie over either, so no load may pass a store (32760 x 1536 RMSNorm with residual
// 72 us with each residual load behind the store before it, 55 us so).
// Not kept, each measured: blocks that loop over rows with the frame's vectors in registers (AdaLN
// 124 us against 79), rows prefetched by cp.async (133 us), four rows a block (110 us): with fewer rows in
// flight the reductions' latency shows.
template <typename T, int MODE, bool WARP, int NE, bool AL, bool FULL>
__global__ void __launch_bounds__(WARP || NE == 16 ? 128 : NE == 24 ? 1024 : NE == 40 ? 256 : 512,
                                  NE == 48 && MODE == QUANT && !WARP ? 2 : 0) row_kernel(const Args p) {
    constexpr int VEC = chunk_values<T, MODE, AL>(), NV = NE / VEC;
    __shared__ float2 red[2][32];
    let_next_start();
    wait_for_earlier();
    Reduce<WARP> reduce{red};
    const int t = WARP ? (int)(threadIdx.x & 31) : (int)threadIdx.x, G = WARP ? 32 : (int)blockDim.x, d = p.d;
    const int64_t row = WARP ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
    if (row >= p.n) return;   // whole warps (WARP); no block barrier follows
    const T *x = static_cast<const T *>(p.x) + row * p.x_ld, *r = static_cast<const T *>(p.res) + row * p.res_ld;
    const T *w = static_cast<const T *>(p.weight), *b = static_cast<const T *>(p.bias);
    const int64_t f = (MODE >= MOD && p.frame_tokens > 0) ? (unsigned)row / (unsigned)p.frame_tokens : 0;
    auto at = [&](int i) { return (i * G + t) * VEC; };
    // A chunk past the row's end loads the row's last chunk again and counts for nothing: not in the sums, and
    // not in the maxima either, because the sum stored over an input may have changed what it read. (Without
    // AL a chunk is filled with zeros past the end.)
    constexpr bool WHOLE = FULL || !AL;   // every chunk counts
    auto from = [&](int i) { return WHOLE ? at(i) : min(at(i), d - VEC); };
    auto in = [&](int i) { return at(i) < d; };
    uint64_t v[NV][VEC / 2];   // pairs of values
    {
        Chunk<T, VEC, AL, FULL> xv[NV], rv[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) xv[i].load(x, from(i), d);
        if (MODE != QUANT && p.res) {
#pragma unroll
            for (int i = 0; i < NV; ++i) rv[i].load(r, from(i), d);
        }
        // The frame's vectors come to L1 while the row is on its way. Warps of wide 16-bit rows only: AdaLN with the
        // gated addition, without and with, 4680 x 1536 17.1 / 13.9 us, 32760 x 1536 68.9 / 61.8 us and 32760 x 1024
        // 48.5 / 46.0 us; slower for 512 values (25.8 / 28.6 us), in blocks (2048 values, 102 / 126 us) and for
        // fp32 (4680 x 1536 19.5 / 20.2 us).
        if (MODE == MOD && WARP && NE > 16 && AL && sizeof(T) == 2 && p.gate) {
            for (int c = (int)threadIdx.x * 32; c < d; c += (int)blockDim.x * 32) {
                prefetch_l1(p.gate + f * p.gate_ld + c);
                prefetch_l1(p.scale + f * p.mod_ld + c);
                prefetch_l1(p.shift + f * p.mod_ld + c);
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) v[i][j] = xv[i][j];
        if (MODE != QUANT && p.res) {
            if (MODE >= MOD && p.gate) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    Chunk<float, VEC, AL, FULL> g;
                    g.load(p.gate + f * p.gate_ld, from(i), d);
#pragma unroll
                    for (int j = 0; j < VEC / 2; ++j) v[i][j] = add_both(v[i][j], f2_mul(rv[i][j], g[j]));
                }
            } else {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < VEC / 2; ++j) v[i][j] = f2_add(v[i][j], rv[i][j]);
            }
            if (p.sum) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    Chunk<T, VEC, AL, FULL> o;
#pragma unroll
                    for (int j = 0; j < VEC / 2; ++j) o.set(j, v[i][j]);
                    o.store(static_cast<T *>(p.sum) + row * p.sum_ld, at(i), d);
                }
            }
        }
    }
    float rstd = 1.f, m = 0.f;
    uint64_t s2 = 0ull;
    uint32_t top;
    if (MODE == QUANT) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float most = WHOLE ? m : 0.f;
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) most = max_abs(max_abs(most, f2_lo(v[i][j])), f2_hi(v[i][j]));
            if (WHOLE) m = most;
            else if (in(i)) m = max_abs(m, most);
        }
        top = reduce.max_bits(__float_as_uint(m));
    } else if (MODE == RMS) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            Chunk<T, VEC, AL, FULL> a;
            a.load(w, from(i), d);
            uint64_t part = WHOLE ? s2 : 0ull;
            float most = WHOLE ? m : 0.f;
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) {
                part = f2_fma(v[i][j], v[i][j], part);
                v[i][j] = f2_mul(v[i][j], a[j]);
                most = max_abs(max_abs(most, f2_lo(v[i][j])), f2_hi(v[i][j]));
            }
            if (WHOLE) {
                s2 = part;
                m = most;
            } else if (in(i)) {
                s2 = f2_add(s2, part);
                m = max_abs(m, most);
            }
        }
        const float2 a = reduce(f2_lo(s2) + f2_hi(s2), __float_as_uint(m));
        rstd = inv_root(a.x * p.inv_d, p.eps);
        top = rstd > 0.f ? __float_as_uint(a.y) : __float_as_uint(rstd);   // the codes are made without it
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            uint64_t part = WHOLE ? s2 : 0ull;
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) part = f2_add(part, v[i][j]);
            if (WHOLE) s2 = part;
            else if (in(i)) s2 = f2_add(s2, part);
        }
        const float mean = reduce.sum(f2_lo(s2) + f2_hi(s2)) * p.inv_d;
        s2 = 0ull;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            uint64_t part = WHOLE ? s2 : 0ull;
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) {
                v[i][j] = f2_add(v[i][j], f2(-mean, -mean));
                if constexpr (!AL)   // past the row's end
                    v[i][j] = f2(at(i) + 2 * j < d ? f2_lo(v[i][j]) : 0.f, at(i) + 2 * j + 1 < d ? f2_hi(v[i][j]) : 0.f);
                part = f2_fma(v[i][j], v[i][j], part);
            }
            if (WHOLE) s2 = part;
            else if (in(i)) s2 = f2_add(s2, part);
        }
        rstd = inv_root(reduce.sum(f2_lo(s2) + f2_hi(s2)) * p.inv_d, p.eps);
        const uint64_t rstd2 = f2(rstd, rstd);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (MODE == AFFINE) {
                Chunk<T, VEC, AL, FULL> a, e;
                a.load(w, from(i), d);
                e.load(b, from(i), d);
#pragma unroll
                for (int j = 0; j < VEC / 2; ++j) v[i][j] = f2_fma(v[i][j], f2_mul(rstd2, a[j]), e[j]);
            } else {
                Chunk<float, VEC, AL, FULL> a, e;
                a.load(p.scale + f * p.mod_ld, from(i), d);
                e.load(p.shift + f * p.mod_ld, from(i), d);
#pragma unroll
                for (int j = 0; j < VEC / 2; ++j) v[i][j] = f2_fma(v[i][j], f2_fma(rstd2, a[j], rstd2), e[j]);
            }
            float most = WHOLE ? m : 0.f;
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) most = max_abs(max_abs(most, f2_lo(v[i][j])), f2_hi(v[i][j]));
            if (WHOLE) m = most;
            else if (in(i)) m = max_abs(m, most);
        }
        top = reduce.max_bits(__float_as_uint(m));
    }
    const Scale q = row_scale(top);
    int8_t *out = p.out + row * p.out_ld;
#pragma unroll
    for (int i = 0; i < NV; ++i) store_codes<VEC, FULL>(out, at(i), d, p.out_words, v[i], q);
    if (t == 0) p.scales[row] = MODE == RMS ? __fmul_rn(q.s, rstd) : q.s;
}

// Rows too long for registers: one CTA per row, element loads, the row read once per statistic. Places in the
// row are unsigned: the step past the end of a row of nearly 2^31 values must not wrap to a negative one.
template <typename T, int MODE>
__global__ void __launch_bounds__(512) long_row_kernel(const Args p) {
    __shared__ float2 red[2][32];
    let_next_start();
    wait_for_earlier();
    Reduce<false> reduce{red};
    const int64_t row = blockIdx.x;
    const unsigned t = threadIdx.x, d = (unsigned)p.d;
    const T *x = static_cast<const T *>(p.x) + row * p.x_ld;
    const T *r = p.res ? static_cast<const T *>(p.res) + row * p.res_ld : nullptr;
    const int64_t f = (MODE >= MOD && p.frame_tokens > 0) ? (unsigned)row / (unsigned)p.frame_tokens : 0;
    const float *g = p.gate ? p.gate + f * p.gate_ld : nullptr;
    const T *w = static_cast<const T *>(p.weight), *b = static_cast<const T *>(p.bias);
    const float *sh = p.shift + f * p.mod_ld, *sc = p.scale + f * p.mod_ld;
    auto value = [&](unsigned c) -> float {
        float v = to_f(x[c]);
        if (r) v = __fadd_rn(v, g ? __fmul_rn(to_f(r[c]), g[c]) : to_f(r[c]));
        return v;
    };
    float mean = 0.f, rstd = 1.f;
    if (MODE == RMS) {
        float s = 0.f;
        for (unsigned c = t; c < d; c += blockDim.x) {
            const float v = value(c);
            s += v * v;
        }
        rstd = inv_root(reduce.sum(s) * p.inv_d, p.eps);
    } else if (MODE >= MOD) {
        float s = 0.f;
        for (unsigned c = t; c < d; c += blockDim.x) s += value(c);
        mean = reduce.sum(s) * p.inv_d;
        s = 0.f;
        for (unsigned c = t; c < d; c += blockDim.x) {
            const float z = value(c) - mean;
            s += z * z;
        }
        rstd = inv_root(reduce.sum(s) * p.inv_d, p.eps);
    }
    auto coded = [&](unsigned c, float v) -> float {   // what the codes stand for, up to RMS's rsqrt
        if (MODE == QUANT) return v;
        if (MODE == RMS) return __fmul_rn(v, to_f(w[c]));
        const float z = (v - mean) * rstd;
        return MODE == AFFINE ? z * to_f(w[c]) + to_f(b[c]) : z * (1.f + sc[c]) + sh[c];
    };
    float m = 0.f;
    for (unsigned c = t; c < d; c += blockDim.x) m = max_abs(m, coded(c, value(c)));
    uint32_t top = reduce.max_bits(__float_as_uint(m));
    if (MODE == RMS && !(rstd > 0.f)) top = __float_as_uint(rstd);
    const Scale s = row_scale(top);
    for (unsigned c = t; c < d; c += blockDim.x) {
        const float v = value(c);
        p.out[row * p.out_ld + c] = (int8_t)code(coded(c, v), s);
        // after the last read of x[c] and r[c], by the thread that read them: the sum may be
        // written over either
        if (p.sum) from_f(v, static_cast<T *>(p.sum)[row * p.sum_ld + c]);
    }
    if (t == 0) p.scales[row] = MODE == RMS ? __fmul_rn(s.s, rstd) : s.s;
}

// The sum where nothing is added: x itself. A kernel of its own, because a store outside the residual's branch
// cost the norms 0.3 to 6 us (registers; 4680 x 1536 AdaLN 8.1 / 8.7 us, 4000 x 8960 RMSNorm 40 / 46 us).
template <typename T>
__global__ void __launch_bounds__(256) copy_kernel(const Args p) {
    let_next_start();
    wait_for_earlier();
    const T *x = static_cast<const T *>(p.x) + (int64_t)blockIdx.x * p.x_ld;
    T *to = static_cast<T *>(p.sum) + (int64_t)blockIdx.x * p.sum_ld;
    for (unsigned c = threadIdx.x; c < (unsigned)p.d; c += blockDim.x) to[c] = x[c];
}

static size_t type_bytes(int dtype) { return dtype == SS_F32 ? 4 : 2; }
static bool off(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

// FULL where every thread's last chunk is in the row, that is where the width is the threads times their
// values: no bounds. 4680 rows of 1536 values with and without: AdaLN 8.1 / 11.6 us, with the gated addition
// 13.8 / 18.5 us, RMSNorm with residual 10.6 / 11.5 us; quantiser of 8960 values 20.5 / 21.3 us.
template <typename T, int MODE, int NE, bool AL>
static void launch_warps(const Args &p, cudaStream_t st) {
    const unsigned blocks = (unsigned)(((int64_t)p.n + 3) / 4);
    if (AL && p.d == 32 * NE) launch_after(row_kernel<T, MODE, true, NE, AL, AL>, blocks, 128, 0, st, 1, p);
    else launch_after(row_kernel<T, MODE, true, NE, AL, false>, blocks, 128, 0, st, 1, p);
}
template <typename T, int MODE, int NE, bool AL>
static void launch_blocks(const Args &p, cudaStream_t st) {
    constexpr int VEC = chunk_values<T, MODE, AL>(), NV = NE / VEC;
    const int chunks = (p.d + VEC - 1) / VEC, threads = ((chunks + NV - 1) / NV + 31) / 32 * 32;
    if (AL && p.d == threads * NE) launch_after(row_kernel<T, MODE, false, NE, AL, AL>, p.n, threads, 0, st, 1, p);
    else launch_after(row_kernel<T, MODE, false, NE, AL, false>, p.n, threads, 0, st, 1, p);
}
// The smallest group whose registers hold the row: a warp up to 1536 values (no block barrier; few
// values a thread for narrow rows: 32760 x 512 RMSNorm with residual 20 us at 16 a thread, 44 at 48; AdaLN
// 28 / 64), blocks after that (2048 values: 69 us at 16 a thread, 74 at 40), and past 24576 values the
// row is read again for each statistic.
template <typename T, int MODE, bool AL>
static int launch_rows(const Args &p, cudaStream_t st) {
    if (AL && p.d <= 32 * 16) launch_warps<T, MODE, AL ? 16 : 48, AL>(p, st);
    else if (AL && p.d <= 32 * 32) launch_warps<T, MODE, AL ? 32 : 48, AL>(p, st);
    else if (p.d <= 32 * 48) launch_warps<T, MODE, 48, AL>(p, st);
    else if (p.d <= 128 * 16) launch_blocks<T, MODE, 16, AL>(p, st);
    else if (p.d <= 256 * 40) launch_blocks<T, MODE, 40, AL>(p, st);
    else if (p.d <= 512 * 48) launch_blocks<T, MODE, sizeof(T) == 4 ? 24 : 48, AL>(p, st);   // registers
    else launch_after(long_row_kernel<T, MODE>, p.n, 512, 0, st, 1, p);
    return (int)cudaGetLastError();
}

template <typename T, int MODE>
static int launch_type(Args p, cudaStream_t st) {
    constexpr int VEC = chunk_values<T, MODE, true>();
    constexpr size_t bytes = VEC * sizeof(T);
    if (p.sum && !p.res) {
        if (p.sum != p.x || p.sum_ld != p.x_ld) {
            const cudaError_t e = launch_after(copy_kernel<T>, (unsigned)p.n, 256, 0, st, 1, p);
            if (e != cudaSuccess) return (int)e;
        }
        p.sum = nullptr;
    }
    // rows and vectors all start at a chunk's boundary and end at a whole chunk
    const bool al = p.d % VEC == 0 && !off(p.x, bytes) && p.x_ld % VEC == 0 && !off(p.weight, bytes) &&
                    !off(p.bias, bytes) && (!p.res || (!off(p.res, bytes) && p.res_ld % VEC == 0)) &&
                    (!p.sum || (!off(p.sum, bytes) && p.sum_ld % VEC == 0)) &&
                    (!p.gate || (!off(p.gate, 16) && p.gate_ld % 4 == 0)) &&
                    (!p.shift || (!off(p.shift, 16) && !off(p.scale, 16) && p.mod_ld % 4 == 0));
    p.inv_d = 1.f / (float)p.d;
    const size_t word = al ? VEC : 4;
    p.out_words = !off(p.out, word) && p.out_ld % (int64_t)word == 0;
    return al ? launch_rows<T, MODE, true>(p, st) : launch_rows<T, MODE, false>(p, st);
}

template <int MODE>
static int launch(const Args &p, int dtype, cudaStream_t st) {
    if (dtype == SS_BF16) return launch_type<__nv_bfloat16, MODE>(p, st);
    if (dtype == SS_F16) return launch_type<__half, MODE>(p, st);
    return launch_type<float, MODE>(p, st);
}

// checks shared by the three entry points; 0 when the call is one the kernels can run
static int check_rows(const Args &p, int dtype) {
    if (dtype != SS_BF16 && dtype != SS_F32 && dtype != SS_F16) return SS_ERR_SHAPE;
    if (p.n < 0 || p.d <= 0 || p.x_ld < p.d || p.out_ld < p.d) return SS_ERR_SHAPE;
    if ((p.res && p.res_ld < p.d) || (p.sum && p.sum_ld < p.d)) return SS_ERR_SHAPE;
    if (p.n == 0) return 0;   // buffers without rows may have no address
    if (!p.x || !p.out || !p.scales) return SS_ERR_POINTER;
    const size_t a = type_bytes(dtype);
    if (off(p.x, a) || off(p.res, a) || off(p.sum, a) || off(p.weight, a) || off(p.bias, a) || off(p.scales, 4) ||
        off(p.gate, 4) || off(p.shift, 4) || off(p.scale, 4))
        return SS_ERR_POINTER;
    return 0;
}

}  // namespace rows
}  // namespace ss

extern "C" int ss_quant_rows(const void *x, int64_t x_ld, int dtype, int n, int d, int8_t *out, int64_t out_ld,
                             float *scales, void *stream) {
    using namespace ss::rows;
    Args p = {};
    p.x = x, p.x_ld = x_ld, p.n = n, p.d = d, p.out = out, p.out_ld = out_ld, p.scales = scales;
    const int rc = check_rows(p, dtype);
    if (rc || n == 0) return rc;
    return launch<QUANT>(p, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int ss_rms_norm_i8(const void *x, int64_t x_ld, const void *residual, int64_t res_ld, int dtype, int n,
                              int d, const void *weight, float eps, void *sum, int64_t sum_ld, int8_t *out,
                              int64_t out_ld, float *scales, void *stream) {
    using namespace ss::rows;
    Args p = {};
    p.x = x, p.x_ld = x_ld, p.res = residual, p.res_ld = res_ld, p.weight = weight, p.eps = eps;
    p.sum = sum, p.sum_ld = sum_ld, p.n = n, p.d = d, p.out = out, p.out_ld = out_ld, p.scales = scales;
    if (!weight) return SS_ERR_POINTER;
    const int rc = check_rows(p, dtype);
    if (rc || n == 0) return rc;
    return launch<RMS>(p, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int ss_adaln_i8(const void *x, int64_t x_ld, const void *y, int64_t y_ld, const float *gate,
                           int64_t gate_ld, int dtype, int n, int d, int frame_tokens, const float *shift,
                           const float *scale, int64_t mod_ld, const void *weight, const void *bias, float eps,
                           void *sum, int64_t sum_ld, int8_t *out, int64_t out_ld, float *scales, void *stream) {
    using namespace ss::rows;
    Args p = {};
    p.x = x, p.x_ld = x_ld, p.res = y, p.res_ld = y_ld, p.gate = gate, p.gate_ld = gate_ld;
    p.shift = shift, p.scale = scale, p.mod_ld = mod_ld, p.weight = weight, p.bias = bias, p.eps = eps;
    p.frame_tokens = frame_tokens, p.sum = sum, p.sum_ld = sum_ld, p.n = n, p.d = d;
    p.out = out, p.out_ld = out_ld, p.scales = scales;
    const bool affine = weight || bias, modulate = shift || scale;
    if (affine == modulate) return SS_ERR_SHAPE;   // exactly one of the two forms
    if ((affine && (!weight || !bias)) || (modulate && (!shift || !scale)) || (gate && !y)) return SS_ERR_POINTER;
    if (((modulate || gate) && frame_tokens <= 0) || (modulate && mod_ld < d) || (gate && gate_ld < d))
        return SS_ERR_SHAPE;
    const int rc = check_rows(p, dtype);
    if (rc || n == 0) return rc;
    return affine ? launch<AFFINE>(p, dtype, static_cast<cudaStream_t>(stream))
                  : launch<MOD>(p, dtype, static_cast<cudaStream_t>(stream));
}
