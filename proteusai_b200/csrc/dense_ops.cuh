// Shared parts of the feed-forward products (dense_tile.cuh): activations and their derivatives, the layout of the
// saved pre-activations, the elementwise half of the backward pass, and the copy that aligns an operand's rows.
//
//   linear   y = act(z) + r,  z = x W^T + b             dz = dy act'(z)
//   gated    h = act(g) u,    g = x Wg^T + bg, u = ...   dg = dh u act'(g), du = dh act(g)
//
// Inputs and outputs are bf16 or fp16; products accumulate in fp32 and everything up to the one rounding of each output is fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace pai {

enum { ACT_NONE = 0, ACT_GELU = 1, ACT_SILU = 2, ACT_RELU = 3, ACT_SIGMOID = 4, ACT_COUNT = 5 };

__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// log2 Phi(n), n <= 0, as a polynomial of degree 7: Chebyshev fit of log2 of the normal distribution function on [-6, 0], so that
// 2^p has a RELATIVE error below 4e-6 there (half a bf16 step is 2^-9 .. 2^-8, half an fp16 step 2^-12 .. 2^-11).  Below -6 it keeps
// falling, where x Phi(x) is below 1e-8 in magnitude: the absolute error of x Phi(x) stays
// below 6e-7 on the whole negative axis.  One SFU operation, against two for the rational form of erfc.  n is cut off at -30, where
// Phi(n) is 0 in fp32, so that infinities do not meet that 0.
#define PAI_PHI_COEFFS                                                                                                    \
    {-9.999943403e-01f, 1.151269147e+00f, -4.584097768e-01f, 5.402068712e-02f, 8.539461332e-03f, 9.388679333e-04f, \
     6.268140101e-05f,  1.889626234e-06f}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Phi(n) for n in [-30, 0]
__device__ __forceinline__ float normal_tail(float n) {
    constexpr float c[8] = PAI_PHI_COEFFS;
    float p = c[7];
#pragma unroll
    for (int i = 6; i >= 0; --i) p = fmaf(p, n, c[i]);
    return ex2_approx(p);
}
// x Phi(x) = max(x, 0) + n Phi(n), n = -min(|x|, 30), for a pair, the polynomial in packed arithmetic
__device__ __forceinline__ void gelu2(float &x0, float &x1) {
    constexpr float c[8] = PAI_PHI_COEFFS;
    const f2_t n = f2_pack(fmaxf(-fabsf(x0), -30.f), fmaxf(-fabsf(x1), -30.f));
    f2_t p = f2_pack(c[7], c[7]);
#pragma unroll
    for (int i = 6; i >= 0; --i) p = f2_fma(p, n, f2_pack(c[i], c[i]));
    float p0, p1;
    f2_unpack(p, p0, p1);
    const f2_t e = f2_pack(ex2_approx(p0), ex2_approx(p1));
    f2_unpack(f2_fma(n, e, f2_pack(max_nan(x0, 0.f), max_nan(x1, 0.f))), x0, x1);
}
__device__ __forceinline__ float sigmoid_f(float x) { return rcp_approx(1.f + ex2_approx(-1.4426950408889634f * x)); }

template <int ACT>
__device__ __forceinline__ void act_pair(float &a, float &b) {
    if (ACT == ACT_GELU) {
        gelu2(a, b);
    } else if (ACT == ACT_SILU) {
        a *= sigmoid_f(a), b *= sigmoid_f(b);
    } else if (ACT == ACT_RELU) {
        a = max_nan(a, 0.f), b = max_nan(b, 0.f);
    } else if (ACT == ACT_SIGMOID) {
        a = sigmoid_f(a), b = sigmoid_f(b);
    }
}

// act(z) and act'(z)
template <int ACT>
__device__ __forceinline__ void act_and_slope(float z, float &a, float &d) {
    if (ACT == ACT_GELU) {
        const float n = fmaxf(-fabsf(z), -30.f), e = normal_tail(n), phi = z < 0.f ? e : 1.f - e;
        a = fmaf(n, e, max_nan(z, 0.f));
        d = fmaf(z * 0.3989422804014327f, ex2_approx(-0.7213475204444817f * z * z), phi);
    } else if (ACT == ACT_SILU) {
        const float s = sigmoid_f(z);
        a = z * s;
        d = s * fmaf(z, 1.f - s, 1.f);
    } else if (ACT == ACT_RELU) {
        a = max_nan(z, 0.f);
        d = z > 0.f ? 1.f : 0.f;
    } else if (ACT == ACT_SIGMOID) {
        a = sigmoid_f(z);
        d = a * (1.f - a);
    } else {
        a = z, d = 1.f;
    }
}

// ---- 16-bit types: `half` != 0 is fp16, 0 is bf16 -----------------------------------------------------------------
__device__ __forceinline__ unsigned short to_bits16(float v, int half) {
    return half ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}
__device__ __forceinline__ float from_bits16(unsigned short b, int half) {
    return half ? __half2float(__ushort_as_half(b)) : __uint_as_float((uint32_t)b << 16);
}
__device__ __forceinline__ uint32_t pack_bits16(float lo, float hi, int half) {
    if (half) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&b);
}
__device__ __forceinline__ void unpack_bits16(uint32_t w, int half, float &lo, float &hi) {
    if (half) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        lo = f.x, hi = f.y;
    } else {
        lo = __uint_as_float(w << 16), hi = __uint_as_float(w & 0xffff0000u);
    }
}

// ---- saved pre-activations ----------------------------------------------------------------------------------------
// What the backward pass needs besides its inputs is z (linear, with an activation) or g and u (gated).  Rounding them to the tensors'
// own 16-bit type would add an error as large as the outputs' rounding, so they are kept in more bits, in blocks of 32 rows x 32 columns:
//   fp32   [piece of 4 columns][row][4]: a thread per row and a thread per column both write whole sectors
//   fp16   (bf16 tensors, dense_pair.cuh) [piece of 8 columns][row][8] with one power of two per row and 16 columns, chosen so that the largest
//          magnitude of the run lies in [2^14, 2^15): 2^-12 relative accuracy for everything within 2^-28 of it, in 16 bits.  The exponents
//          (int8, [block][half][row]) follow the values.
__host__ __device__ inline size_t saved_blocks(long long rows, int cols) { return (size_t)((rows + 31) / 32) * (size_t)((cols + 31) / 32); }
__host__ __device__ inline size_t saved_bytes_f32(long long rows, int cols) { return saved_blocks(rows, cols) * 4096; }
__host__ __device__ inline size_t saved_bytes_f16(long long rows, int cols) { return saved_blocks(rows, cols) * (2048 + 64); }
__device__ __forceinline__ size_t saved_block(long long row, int col, int col_blocks) { return (size_t)(row >> 5) * col_blocks + (col >> 5); }
__device__ __forceinline__ size_t saved_index_f32(long long row, int col, int col_blocks) {
    return (saved_block(row, col, col_blocks) * 8 + ((col & 31) >> 2)) * 128 + (size_t)(row & 31) * 4 + (col & 3);
}
// eight columns (col a multiple of 8) of a row: the loads, and the values from what they brought
template <bool F32>
struct Saved8 {
    uint4 v[F32 ? 2 : 1];
    int e;
    __device__ __forceinline__ void load(const uint8_t *save, size_t exps, long long row, int col, int col_blocks) {
        const size_t block = saved_block(row, col, col_blocks);
        if (F32) {
            const uint4 *src = reinterpret_cast<const uint4 *>(save + block * 4096) + ((col & 31) >> 2) * 32 + (row & 31);
            v[0] = src[0], v[F32 ? 1 : 0] = src[32];
        } else {
            v[0] = reinterpret_cast<const uint4 *>(save + block * 2048)[((col & 31) >> 3) * 32 + (row & 31)];
            e = reinterpret_cast<const signed char *>(save)[exps + block * 64 + ((col & 31) >> 4) * 32 + (row & 31)];
        }
    }
    __device__ __forceinline__ void get(float (&z)[8]) const {
        const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[F32 ? 1 : 0].x, v[F32 ? 1 : 0].y, v[F32 ? 1 : 0].z, v[F32 ? 1 : 0].w};
        if (F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = __uint_as_float(w[i]);
        } else {
            const float s = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                unpack_bits16(w[i], 1, z[2 * i], z[2 * i + 1]);
                z[2 * i] *= s, z[2 * i + 1] *= s;
            }
        }
    }
};

// ---- elementwise half of the backward pass ------------------------------------------------------------------------
// One warp covers 8 rows x 32 columns a step (4 lanes x 8 columns per row), a CTA 8 rows x 256 columns; it walks down a strip of
// `strip` rows, two steps' loads in flight, and keeps the column sums of what it writes in registers (the bias gradients), joined over the
// eight row lanes by shuffles and written as one partial row per strip; dense_colsum adds the strips.  HBM-bound: gated in bf16 reads dh, g, u and writes dg, du, 10 bytes per element.
struct DenseBwdElemParams {
    const unsigned short *dy;
    long long ld_dy;
    const uint8_t *save0, *save1;   // z, or g and u
    size_t save_exps;               // fp16 form: offset of the exponents
    unsigned short *d0, *d1;        // dz, or dg and du; NULL: not wanted
    long long ld_d;
    float *part0, *part1;           // [strips, N] column sums, or NULL
    long long M;
    int N, strip, vec_dy;
};

template <bool DUAL, int ACT, int HALF, bool F32>
__global__ void __launch_bounds__(256) dense_bwd_elem_kernel(const __grid_constant__ DenseBwdElemParams p) {
    pdl_trigger();
    pdl_wait();
    constexpr bool PLAIN = !DUAL && ACT == ACT_NONE;  // sums of dy alone
    constexpr int U = 2;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c0 = blockIdx.x * 256 + warp * 32 + (lane & 3) * 8;
    const long long r_begin = (long long)blockIdx.y * p.strip;
    const long long r_end = r_begin + p.strip < p.M ? r_begin + p.strip : p.M;
    const int col_blocks = (p.N + 31) >> 5;
    float s0[8], s1[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s0[i] = s1[i] = 0.f;
    const int nc = p.N - c0;  // columns of this thread that exist (may be <= 0 or > 8)
    if (nc > 0) {
        const bool vec = p.vec_dy && nc >= 8;
        for (long long r0 = r_begin + (lane >> 2); r0 < r_end; r0 += 8 * U) {
            uint32_t w[U][4];
            Saved8<F32> z[U], u[U];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const long long r = r0 + 8 * k;
                if (r < r_end) {
                    const unsigned short *src = p.dy + r * p.ld_dy + c0;
                    if (vec) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(src);
                        w[k][0] = v.x, w[k][1] = v.y, w[k][2] = v.z, w[k][3] = v.w;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            w[k][i] = (2 * i < nc ? (uint32_t)src[2 * i] : 0u) | (2 * i + 1 < nc ? (uint32_t)src[2 * i + 1] << 16 : 0u);
                    }
                    if (!PLAIN) z[k].load(p.save0, p.save_exps, r, c0, col_blocks);
                    if (DUAL) u[k].load(p.save1, p.save_exps, r, c0, col_blocks);
                }
            }
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const long long r = r0 + 8 * k;
                if (r < r_end) {
                    float o0[8], o1[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) unpack_bits16(w[k][i], HALF, o0[2 * i], o0[2 * i + 1]);
                    if (!PLAIN) {
                        float zz[8], uu[8];
                        z[k].get(zz);
                        if (DUAL) u[k].get(uu);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            float a, d;
                            act_and_slope<ACT>(zz[i], a, d);
                            if (DUAL) o1[i] = o0[i] * a, d *= uu[i];
                            o0[i] *= d;
                        }
                    }
                    // (columns past N: dy is 0 there but z is not defined; their sums are never stored)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        s0[i] += o0[i];
                        if (DUAL) s1[i] += o1[i];
                    }
                    if (!PLAIN && p.d0) {  // rows of d0 / d1 are padded to a multiple of 8 columns: whole 16-byte words, the tail is never read
                        *reinterpret_cast<uint4 *>(p.d0 + r * p.ld_d + c0) = make_uint4(pack_bits16(o0[0], o0[1], HALF), pack_bits16(o0[2], o0[3], HALF),
                                                                                       pack_bits16(o0[4], o0[5], HALF), pack_bits16(o0[6], o0[7], HALF));
                        if (DUAL)
                            *reinterpret_cast<uint4 *>(p.d1 + r * p.ld_d + c0) =
                                make_uint4(pack_bits16(o1[0], o1[1], HALF), pack_bits16(o1[2], o1[3], HALF), pack_bits16(o1[4], o1[5], HALF),
                                           pack_bits16(o1[6], o1[7], HALF));
                    }
                }
            }
        }
    }
    if (p.part0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                s0[i] += __shfl_xor_sync(0xffffffffu, s0[i], o);
                if (DUAL) s1[i] += __shfl_xor_sync(0xffffffffu, s1[i], o);
            }
        }
        if (lane < 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < nc) {
                    p.part0[(size_t)blockIdx.y * p.N + c0 + i] = s0[i];
                    if (DUAL && p.part1) p.part1[(size_t)blockIdx.y * p.N + c0 + i] = s1[i];
                }
        }
    }
}

// ---- bias gradients: out[c] = sum over strips of part[s, c] -------------------------------------------------------
// The product that follows the elementwise pass does it with a warp that has nothing else to do (a launch of its own would cost a small backward
// pass several microseconds of host time); dense_colsum_kernel where no product follows.  Lane: a column; sixteen partial sums over the strips
// s = i mod 16, added in order of i: the same bits wherever it runs.
struct DenseColsum {
    const float *part[2];  // NULL: none
    void *out[2];
    int N, strips, fp32;
};

template <int HALF>
__device__ __forceinline__ void dense_colsum(const DenseColsum &c, int warp, int warps) {
    const int lane = threadIdx.x & 31;
    for (int m = 0; m < 2; ++m) {
        if (!c.part[m]) continue;
        for (int col = warp * 32 + lane; col < c.N; col += warps * 32) {
            constexpr int U = 16;
            float s[U];
#pragma unroll
            for (int k = 0; k < U; ++k) s[k] = 0.f;
            for (int i = 0; i < c.strips; i += U)
#pragma unroll
                for (int k = 0; k < U; ++k)
                    if (i + k < c.strips) s[k] += c.part[m][(size_t)(i + k) * c.N + col];
            float sum = s[0];
#pragma unroll
            for (int k = 1; k < U; ++k) sum += s[k];
            if (c.fp32) reinterpret_cast<float *>(c.out[m])[col] = sum;
            else reinterpret_cast<unsigned short *>(c.out[m])[col] = to_bits16(sum, HALF);
        }
    }
}

template <int HALF>
__global__ void __launch_bounds__(32) dense_colsum_kernel(const __grid_constant__ DenseColsum c) {
    pdl_trigger();
    pdl_wait();
    dense_colsum<HALF>(c, (int)blockIdx.x, (int)gridDim.x);
}

// dst[r, 0 .. cols) = src[r, 0 .. cols) for rows of any alignment (TMA wants 16-byte aligned ones), up to three matrices in a launch
constexpr int DENSE_MAX_COPIES = 3;
struct DenseCopyParams {
    const unsigned short *src[DENSE_MAX_COPIES];
    unsigned short *dst[DENSE_MAX_COPIES];
    long long ld_src[DENSE_MAX_COPIES], ld_dst[DENSE_MAX_COPIES], rows[DENSE_MAX_COPIES];
    int cols[DENSE_MAX_COPIES];
};
__global__ void __launch_bounds__(256) dense_copy_rows_kernel(const __grid_constant__ DenseCopyParams p) {
    pdl_trigger();
    pdl_wait();
    const int m = blockIdx.y, cols = p.cols[m], words = (cols + 7) >> 3;
    const long long n = p.rows[m] * words, stride = (long long)gridDim.x * 256;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += stride) {
        const long long r = i / words;
        const int c = (int)(i - r * words) * 8;
        const unsigned short *s = p.src[m] + r * p.ld_src[m] + c;
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t lo = c + 2 * k < cols ? s[2 * k] : 0, hi = c + 2 * k + 1 < cols ? s[2 * k + 1] : 0;
            w[k] = lo | hi << 16;
        }
        *reinterpret_cast<uint4 *>(p.dst[m] + r * p.ld_dst[m] + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

}  // namespace pai
