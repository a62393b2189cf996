// dense_vec_kernel: the forward products for up to eight tokens (decoding), y[t, f] = epilogue( sum_k W[f, k] x[t, k] ).
//
// Bound by reading W once: no tensor core, no staging, no cluster.  A warp takes two rows of W (linear: two neighbouring outputs; gated: the rows of
// Wg and Wu of one output), its lanes 16 bytes each of 256 columns at a time with U steps in flight, keeps 2 TT sums per lane in fp32 and
// joins them by shuffles.  x (a few KB) comes from L1 after its first use in the SM.  One token, 512 -> 2048: 2.5 us, against 6.9 with the tile
// kernel and its reduction split over a cluster.
#pragma once
#include "dense_ops.cuh"

namespace pai {

constexpr int DV_WARPS = 4;
constexpr int DV_MAX_TOKENS = 8;

struct DenseVecParams {
    const unsigned short *x, *w0, *w1;
    const void *bias0, *bias1;
    const unsigned short *residual;
    unsigned short *out;
    float *save0, *save1;
    long long ld_x, ld_w0, ld_w1, ld_out, ld_res;
    int T, N, K, bias_fp32;
};

template <bool DUAL, int ACT, int TT, int HALF>
__global__ void __launch_bounds__(DV_WARPS * 32) dense_vec_kernel(const __grid_constant__ DenseVecParams p) {
    pdl_trigger();
    pdl_wait();
    constexpr int U = TT <= 2 ? 4 : 2;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int f = ((int)blockIdx.x * DV_WARPS + warp) * (DUAL ? 1 : 2);
    if (f >= p.N) return;
    // the two rows of W; past the last output the last one again (its sum is not stored)
    const unsigned short *wa = p.w0 + (long long)f * p.ld_w0;
    const unsigned short *wb = DUAL ? p.w1 + (long long)f * p.ld_w1 : p.w0 + (long long)(f + 1 < p.N ? f + 1 : f) * p.ld_w0;
    // what the epilogue needs of this lane: token t, column fo (linear: lanes 0 .. 2 TT - 1, gated: 0 .. TT - 1)
    const int t = DUAL ? lane : lane >> 1, fo = DUAL ? f : f + (lane & 1);
    const bool mine = t < p.T && t < TT && fo < p.N;
    float b0 = 0.f, b1 = 0.f, r = 0.f;
    if (mine) {
        if (p.bias0) b0 = p.bias_fp32 ? reinterpret_cast<const float *>(p.bias0)[fo] : from_bits16(reinterpret_cast<const unsigned short *>(p.bias0)[fo], HALF);
        if (DUAL && p.bias1) b1 = p.bias_fp32 ? reinterpret_cast<const float *>(p.bias1)[fo] : from_bits16(reinterpret_cast<const unsigned short *>(p.bias1)[fo], HALF);
        if (p.residual) r = from_bits16(p.residual[(long long)t * p.ld_res + fo], HALF);
    }
    float s[2][TT];
#pragma unroll
    for (int i = 0; i < TT; ++i) s[0][i] = s[1][i] = 0.f;
    auto step = [&](const uint4 &a, const uint4 &b, const uint4 (&xs)[TT]) {
        float fa[8], fb[8];
        const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            unpack_bits16(aw[i], HALF, fa[2 * i], fa[2 * i + 1]);
            unpack_bits16(bw[i], HALF, fb[2 * i], fb[2 * i + 1]);
        }
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            const uint32_t xw[4] = {xs[j].x, xs[j].y, xs[j].z, xs[j].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x0, x1;
                unpack_bits16(xw[i], HALF, x0, x1);
                s[0][j] = fmaf(fa[2 * i + 1], x1, fmaf(fa[2 * i], x0, s[0][j]));
                s[1][j] = fmaf(fb[2 * i + 1], x1, fmaf(fb[2 * i], x0, s[1][j]));
            }
        }
    };
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const int whole = p.K & ~7;  // columns in whole 16-byte words
#pragma unroll 1
    for (int k0 = lane * 8; k0 < whole; k0 += 256 * U) {
        uint4 a[U], b[U], xs[U][TT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + 256 * u;
            const bool in = k < whole;
            a[u] = in ? __ldg(reinterpret_cast<const uint4 *>(wa + k)) : zero;
            b[u] = in ? __ldg(reinterpret_cast<const uint4 *>(wb + k)) : zero;
#pragma unroll
            for (int j = 0; j < TT; ++j) xs[u][j] = in && j < p.T ? __ldg(reinterpret_cast<const uint4 *>(p.x + (long long)j * p.ld_x + k)) : zero;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) step(a[u], b[u], xs[u]);
    }
    if (lane < p.K - whole) {  // the last columns of a width that is no multiple of 8, one per lane
        const int k = whole + lane;
        const float fa = from_bits16(wa[k], HALF), fb = from_bits16(wb[k], HALF);
#pragma unroll
        for (int j = 0; j < TT; ++j)
            if (j < p.T) {
                const float xv = from_bits16(p.x[(long long)j * p.ld_x + k], HALF);
                s[0][j] = fmaf(fa, xv, s[0][j]);
                s[1][j] = fmaf(fb, xv, s[1][j]);
            }
    }
#pragma unroll
    for (int j = 0; j < TT; ++j)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            s[0][j] += __shfl_xor_sync(0xffffffffu, s[0][j], o);
            s[1][j] += __shfl_xor_sync(0xffffffffu, s[1][j], o);
        }
    float v0 = 0.f, v1 = 0.f;
#pragma unroll
    for (int j = 0; j < TT; ++j)
        if (j == t) v0 = DUAL || !(lane & 1) ? s[0][j] : s[1][j], v1 = s[1][j];
    if (!mine) return;
    v0 += b0, v1 += b1;
    if (p.save0) {
        const size_t at = saved_index_f32(t, fo, (p.N + 31) >> 5);
        p.save0[at] = v0;
        if (DUAL) p.save1[at] = v1;
    }
    float other = 0.f;
    act_pair<ACT>(v0, other);
    p.out[(long long)t * p.ld_out + fo] = to_bits16((DUAL ? v0 * v1 : v0) + r, HALF);
}

}  // namespace pai
