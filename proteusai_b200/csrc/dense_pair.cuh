// dense_pair_kernel: the products of the feed-forward block at sizes that fill the GPU.  out[t, f] = epilogue( sum_r A[t, r] B[f, r] ),
// one output tile of 256 t x bn f per CTA PAIR: tcgen05.mma.cta_group::2 (M = 256), each CTA of the pair staging its own 128 rows of A and
// half of B, so that a 64-wide reduction block costs each SM 32 KB from L2 per 512 tensor cycles at bn = 256 (64 bytes a cycle; single-CTA tiles of
// 128 x 128 need twice that and were bound by it).  Persistent: the pairs walk the tiles, the accumulator in tensor memory is doubled, and the
// epilogue of one tile runs under the products of the next.
//
// An accumulator lane is an output ROW here (the operands of dense_tile.cuh swapped): a thread of the epilogue holds runs of 32 columns, packs
// them to 16-byte words, and the tile leaves through shared memory by TMA stores (32 columns x 32 rows per warp and step).
//     forward  t = token,           f = output feature, r = input feature:  A = x  (K-major),  B = W (K-major)
//     gated    the same with B = 128 rows of Wg (staged by the pair's first CTA) and 128 of Wu (by its second): columns [0, 128) of the
//              accumulator are g, [128, 256) are u
//     dx       t = token,           f = input feature,  r = output feature: A = dz (K-major),  B = W (MN-major); gated: two pairs in sequence
//     dW       t = output feature,  f = input feature,  r = token:          A = dz (MN-major), B = x (MN-major); the long reduction split
//              over pairs that leave fp32 tiles in the workspace, added in order by dense_reduce_kernel
//
// Warps: 0 TMA loads, 1 MMAs (first CTA of the pair), 2 tensor memory, 3 what is left of the bias gradients, 4..19 epilogue (four per quarter of
// the lanes, a quarter of the columns each; eight with twice the columns and registers took 178 us for 148 with GELU at 65536 x 512 x 2048).
#pragma once
#include "dense_tile.cuh"

namespace pai {

constexpr int DP_BK = 64;  // reduction block: 128 bytes, one swizzle row
constexpr int DP_STAGES = 5;
constexpr int DP_STAGE_BYTES = 32768;  // A 128 x 128 bytes, B up to 128 x 128 bytes
constexpr int DP_EPI_WARPS = 16;
constexpr int DP_THREADS = 128 + 32 * DP_EPI_WARPS;

struct DensePairSmem {
    uint8_t stage[DP_STAGES][DP_STAGE_BYTES];
    uint8_t panel[DP_EPI_WARPS][2][2048];  // per epilogue warp two of 32 rows x 32 columns (64-byte swizzle): residual in, output out
    float bias[2][256];
    uint64_t full[DP_STAGES], free[DP_STAGES], acc_full[2], acc_free[2];
    uint64_t res_full[DP_EPI_WARPS][2];
    uint32_t tmem;
    int abort_flag;
};

enum { DP_LINEAR = 0, DP_GATED = 1, DP_PARTIAL = 2 };
// What an instance of the kernel does beside its products; without DP_ANY the output (and the residual) go by TMA and the flags are all there is, which
// takes the epilogue of 65536 x 512 x 2048 with GELU from 127 to 114 us; DP_ANY looks at its parameters.
enum { DP_RESIDUAL = 1, DP_SAVE = 2, DP_ANY = 4 };

struct DensePairParams {
    unsigned short *out0;
    const unsigned short *residual;
    const void *bias0, *bias1;
    uint8_t *save0, *save1;          // saved pre-activations of g / z and u, or NULL
    float *part;                     // DP_PARTIAL: fp32 tiles, [split][group] matrices in the layout of saved_index_f32
    long long ld_out, ld_res, save_exps;
    int T, F, bn;                    // bn: accumulator columns of a tile (gated: bn / 2 of each)
    int t_tiles, f_tiles, groups, splits;
    int kb_seg, kb_total;
    int a_mn, b_mn, act, bias_fp32;
    int tma_out, tma_res, save_f32;
    uint32_t idesc;
    DenseColsum colsum;              // bias gradients to finish beside the product
};

// ---- CTA-pair forms of the helpers in tc.cuh --------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Byte offset of the 16-byte chunk `chunk` (0..3) of row `row` inside a [rows x 64 B] tile stored with the 64-byte swizzle.
__device__ __forceinline__ uint32_t sw64_offset(int row, int chunk) { return (uint32_t)(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4)); }
// load into this CTA's shared memory, completion on a barrier of either CTA of the pair (`bar`: shared::cluster address)
__device__ __forceinline__ void tma_load_2d_pair(void *dst_smem, const CUtensorMap *map, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
            smem_u32(dst_smem)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, const void *src_smem, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)),
                 "r"(smem_u32(src_smem)), "r"(c0), "r"(c1)
                 : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait_read() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void umma_ss_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// the MMAs issued so far arrive on the barrier at this offset in both CTAs
__device__ __forceinline__ void umma_commit_pair(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                 "h"((unsigned short)3)
                 : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// ---- epilogue -------------------------------------------------------------------------------------------------------
// v[i]: 16 columns (from `col`, a multiple of 16) of row `row` of a block of saved pre-activations; NaN and infinities keep their kind
__device__ __forceinline__ void save_run_f16(uint8_t *values, uint8_t *exps, size_t block, int col, int row, const float *v) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(v[i]));
    if (m > 3.4e38f) {  // an infinity does not set the scale of the others
        m = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) m = isinf(v[i]) ? m : fmaxf(m, fabsf(v[i]));
    }
    int e = (int)(__float_as_uint(m) >> 23) - 127 - 14;  // 2^e 2^14 <= m < 2^e 2^15
    if (m == 0.f) e = 0;
    e = e < -112 ? -112 : e;  // (2^-e stays finite; what is smaller than 2^-98 loses bits)
    const float s = __uint_as_float((uint32_t)(127 - e) << 23);
    uint4 *dst = reinterpret_cast<uint4 *>(values + block * 2048) + ((col & 31) >> 3) * 32 + row;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_bits16(v[q * 8 + 2 * i] * s, v[q * 8 + 2 * i + 1] * s, 1);
        dst[q * 32] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    exps[block * 64 + ((col & 31) >> 4) * 32 + row] = (uint8_t)(signed char)e;
}
__device__ __forceinline__ void save_run_f32(float *values, size_t block, int col, int row, const float *v) {
    float4 *dst = reinterpret_cast<float4 *>(values + block * 1024) + ((col & 31) >> 2) * 32 + row;
#pragma unroll
    for (int q = 0; q < 4; ++q) dst[q * 32] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
}
// The tiles of a pair in turn: every pairs-th in the order (f fastest, t, group, split), so that the pairs of a moment share rows of A and columns of
// B in L2 (a run of neighbours per pair instead: 16384 x 4096 x 4096 takes 449 us for 341, a short reduction the same).  Stepping adds the
// digits of `pairs` with carries: a division per tile would cost the thread that issues the products several hundred cycles between tiles.
struct DensePairTiles {
    int f, t, gs, left;       // digits of the current item (gs = split * groups + group); items left, this one included
    int step_f, step_t, step_gs;
    __device__ __forceinline__ DensePairTiles(const DensePairParams &p, int pair, int pairs) {
        const int items = p.f_tiles * p.t_tiles * p.groups * p.splits, rest = items % pairs;
        left = items / pairs + (pair < rest ? 1 : 0);
        f = pair % p.f_tiles, t = pair / p.f_tiles, gs = t / p.t_tiles, t %= p.t_tiles;
        step_f = pairs % p.f_tiles, step_t = pairs / p.f_tiles, step_gs = step_t / p.t_tiles, step_t %= p.t_tiles;
    }
    __device__ __forceinline__ bool valid() const { return left > 0; }
    __device__ __forceinline__ void next(const DensePairParams &p) {
        --left;
        f += step_f, t += step_t, gs += step_gs;
        if (f >= p.f_tiles) f -= p.f_tiles, ++t;
        if (t >= p.t_tiles) t -= p.t_tiles, ++gs;
    }
    __device__ __forceinline__ int group(const DensePairParams &p) const { return p.groups == 2 ? gs & 1 : 0; }
    __device__ __forceinline__ int split(const DensePairParams &p) const { return p.groups == 2 ? gs >> 1 : gs; }
    // reduction blocks [k0, k1) of the item
    __device__ __forceinline__ void range(const DensePairParams &p, int &k0, int &k1) const {
        k0 = 0, k1 = p.kb_total;
        if (p.splits > 1) {
            const int s = split(p);
            k0 = (int)((long long)p.kb_total * s / p.splits), k1 = (int)((long long)p.kb_total * (s + 1) / p.splits);
        }
    }
};

// 16 columns (from `c` of a 32-column panel): saved pre-activations, activation, product, residual, rounding, into the panel.
template <int MODE, int ACT, int HALF, int FLAGS>
__device__ __forceinline__ void dense_pair_run(const DensePairParams &p, float *v, float *u, bool has_res, uint8_t *panel, int c, int col, size_t block) {
    const int lane = threadIdx.x & 31;
    if ((FLAGS & DP_ANY) ? p.save0 != nullptr : (FLAGS & DP_SAVE) != 0) {
        if ((FLAGS & DP_ANY) ? p.save_f32 != 0 : HALF != 0) {
            save_run_f32(reinterpret_cast<float *>(p.save0), block, col, lane, v);
            if (MODE == DP_GATED) save_run_f32(reinterpret_cast<float *>(p.save1), block, col, lane, u);
        } else {
            save_run_f16(p.save0, p.save0 + p.save_exps, block, col, lane, v);
            if (MODE == DP_GATED) save_run_f16(p.save1, p.save1 + p.save_exps, block, col, lane, u);
        }
    }
#pragma unroll
    for (int i = 0; i < 16; i += 2) act_pair<ACT>(v[i], v[i + 1]);
    if (MODE == DP_GATED) {
#pragma unroll
        for (int i = 0; i < 16; i += 2) f2_unpack(f2_mul(f2_pack(v[i], v[i + 1]), f2_pack(u[i], u[i + 1])), v[i], v[i + 1]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint4 *at = reinterpret_cast<uint4 *>(panel + sw64_offset(lane, (c >> 3) + h));
        if (has_res) {
            const uint4 r = *at;
            const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float lo, hi;
                unpack_bits16(w[i], HALF, lo, hi);
                v[h * 8 + 2 * i] += lo, v[h * 8 + 2 * i + 1] += hi;
            }
        }
        *at = make_uint4(pack_bits16(v[h * 8], v[h * 8 + 1], HALF), pack_bits16(v[h * 8 + 2], v[h * 8 + 3], HALF),
                         pack_bits16(v[h * 8 + 4], v[h * 8 + 5], HALF), pack_bits16(v[h * 8 + 6], v[h * 8 + 7], HALF));
    }
}

// Epilogue of one warp: 32 rows x half of the tile's columns, in panels of 32 columns that alternate between two buffers: while one is
// computed the other leaves by its TMA store, and the residual of the next panel is on its way into it as soon as that store has read it.
// The accumulators of the next step are on their way from tensor memory while a step (32 columns, or 16 of each of two) is computed: beside
// running products a tcgen05.ld takes most of a thousand cycles.
template <int MODE, int ACT, int HALF, int FLAGS>
__device__ __forceinline__ void dense_pair_epilogue(const DensePairParams &p, DensePairSmem &sm, const CUtensorMap *my, const CUtensorMap *mr,
                                                    uint32_t tmem, uint32_t rank, DensePairTiles t) {
    constexpr int STEP = MODE == DP_GATED ? 16 : 32, GROUPS = DP_EPI_WARPS / 4;
    const int ew = (threadIdx.x >> 5) - 4, lane = threadIdx.x & 31, q = ew & 3, g = ew >> 2;
    const int f_width = MODE == DP_GATED ? p.bn / 2 : p.bn, panels = f_width / (32 * GROUPS);  // panels of this warp per tile: 4 or 2
    const int col_blocks = (p.F + 31) >> 5;
    const uint32_t acc_free0 = map_to_rank(smem_u32(&sm.acc_free[0]), 0), acc_free1 = map_to_rank(smem_u32(&sm.acc_free[1]), 0);
    const bool has_res = MODE == DP_LINEAR && ((FLAGS & DP_ANY) ? p.residual != nullptr : (FLAGS & DP_RESIDUAL) != 0);
    const bool res_tma = has_res && (!(FLAGS & DP_ANY) || p.tma_res), out_tma = !(FLAGS & DP_ANY) || p.tma_out;
    const bool has_bias = MODE != DP_PARTIAL && (p.bias0 || (MODE == DP_GATED && p.bias1));
    auto row_of = [&](const DensePairTiles &x) { return x.t * 256 + (int)rank * 128 + q * 32; };
    auto col_of = [&](const DensePairTiles &x, int i) { return x.f * f_width + (g * panels + i) * 32; };
    auto fetch_residual = [&](const DensePairTiles &x, int i, int b) {  // (one lane)
        if (row_of(x) < p.T && col_of(x, i) < p.F) {
            mbar_expect_tx(&sm.res_full[ew][b], 2048);
            tma_load_2d(sm.panel[ew][b], mr, col_of(x, i), row_of(x), &sm.res_full[ew][b]);
        }
    };
    // this lane's biases (column lane of each panel) as they are in memory, fetched a tile ahead and converted when used
    uint32_t b0[4] = {0, 0, 0, 0}, b1[2] = {0, 0};
    auto raw_bias = [&](const void *b, int c) -> uint32_t {
        if (!b || c >= p.F) return 0;
        return p.bias_fp32 ? reinterpret_cast<const uint32_t *>(b)[c] : reinterpret_cast<const unsigned short *>(b)[c];
    };
    auto to_bias = [&](uint32_t r) { return p.bias_fp32 ? __uint_as_float(r) : from_bits16((unsigned short)r, HALF); };
    auto fetch_biases = [&](const DensePairTiles &x) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < panels) {
                b0[i] = raw_bias(p.bias0, col_of(x, i) + lane);
                if (MODE == DP_GATED && i < 2) b1[i] = raw_bias(p.bias1, col_of(x, i) + lane);
            }
    };
    if (has_bias) fetch_biases(t);
    if (res_tma && lane == 0) {
        fetch_residual(t, 0, 0);
        if (panels > 1) fetch_residual(t, 1, 1);
    }
    uint32_t res_phase = 0;  // bit b: phase of res_full[b]
    int used = 0;            // panels so far
    for (int n = 0; t.valid(); ++n) {
        const int row0 = row_of(t), a = n & 1;
        DensePairTiles next = t;
        next.next(p);
        if (has_res && !res_tma) {  // any alignment: a row at a time, a column per lane, both panels (at most two) before the products are done
            if (lane == 0) bulk_wait_read<0>();
            __syncwarp();
            for (int i = 0; i < panels; ++i) {
                const int col = col_of(t, i) + lane, rows = p.T - row0;
                uint8_t *panel = sm.panel[ew][(used + i) & 1];
                const unsigned short *src = p.residual + (long long)row0 * p.ld_res + col;
                unsigned short w[32];
#pragma unroll
                for (int r = 0; r < 32; ++r) w[r] = r < rows && col < p.F ? src[(long long)r * p.ld_res] : (unsigned short)0;
#pragma unroll
                for (int r = 0; r < 32; ++r) *reinterpret_cast<unsigned short *>(panel + sw64_offset(r, lane >> 3) + (lane & 7) * 2) = w[r];
            }
            __syncwarp();
        }
        if (!mbar_wait_abortable(&sm.acc_full[a], (n >> 1) & 1, &sm.abort_flag)) break;
        tc_fence_after();
        const uint32_t acc = tmem + a * 256 + ((uint32_t)(q * 32) << 16) + g * panels * 32;
        uint32_t raw[STEP], raw2[MODE == DP_GATED ? STEP : 1];
        auto fetch_acc = [&](int c) {
            if constexpr (MODE == DP_GATED) {
                tmem_ld16(acc + c, raw);
                tmem_ld16(acc + f_width + c, raw2);
            } else {
                tmem_ld32(acc + c, raw);
            }
        };
        // The four warps of a column group write the same biases to the same place.  Nobody still reads this buffer: the accumulator of tile n
        // became full only after every warp had released tile n - 2.
        float *bias = &sm.bias[a][g * panels * 32], *bias2 = &sm.bias[a][128 + g * panels * 32];
        if (has_bias) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < panels) {
                    bias[i * 32 + lane] = to_bias(b0[i]);
                    if (MODE == DP_GATED && i < 2) bias2[i * 32 + lane] = to_bias(b1[i]);
                }
            if (next.valid()) fetch_biases(next);
            __syncwarp();
        }
#pragma unroll 1
        for (int c = 0; c < panels * 32; c += STEP) {
            const int i = c >> 5, col = col_of(t, i), b = used & 1;
            const bool live = row0 < p.T && col < p.F;  // (warp-uniform)
            const bool first = (c & 31) == 0, last = ((c + STEP) & 31) == 0;
            uint8_t *panel = sm.panel[ew][b];
            if (MODE != DP_PARTIAL && first) {
                if (has_res && !res_tma) {  // (the panel holds the residual already)
                } else if (res_tma) {
                    if (live) {
                        mbar_wait_abortable(&sm.res_full[ew][b], (res_phase >> b) & 1, &sm.abort_flag);
                        res_phase ^= 1u << b;
                    }
                } else {
                    if (lane == 0) bulk_wait_read<1>();  // the store before the last one has read this buffer
                    __syncwarp();
                }
            }
            float v[STEP], u[MODE == DP_GATED ? STEP : 1];
            fetch_acc(c);
            tmem_wait_ld();
            if (has_bias) {
#pragma unroll
                for (int k = 0; k < STEP; k += 4) {
                    const float4 w = *reinterpret_cast<const float4 *>(bias + c + k);
                    f2_unpack(f2_add(f2_pack(__uint_as_float(raw[k]), __uint_as_float(raw[k + 1])), f2_pack(w.x, w.y)), v[k], v[k + 1]);
                    f2_unpack(f2_add(f2_pack(__uint_as_float(raw[k + 2]), __uint_as_float(raw[k + 3])), f2_pack(w.z, w.w)), v[k + 2], v[k + 3]);
                    if constexpr (MODE == DP_GATED) {
                        const float4 x = *reinterpret_cast<const float4 *>(bias2 + c + k);
                        f2_unpack(f2_add(f2_pack(__uint_as_float(raw2[k]), __uint_as_float(raw2[k + 1])), f2_pack(x.x, x.y)), u[k], u[k + 1]);
                        f2_unpack(f2_add(f2_pack(__uint_as_float(raw2[k + 2]), __uint_as_float(raw2[k + 3])), f2_pack(x.z, x.w)), u[k + 2], u[k + 3]);
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < STEP; ++k) {
                    v[k] = __uint_as_float(raw[k]);
                    if constexpr (MODE == DP_GATED) u[k] = __uint_as_float(raw2[k]);
                }
            }
            if (c + STEP == panels * 32) {  // the accumulator has been read: the products may have it back
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(a ? acc_free1 : acc_free0);
            }
            const size_t block = saved_block(row0, col, col_blocks);
            if (MODE == DP_PARTIAL) {
                if (live) {
                    float *part = p.part + (size_t)t.gs * (saved_bytes_f32(p.T, p.F) / 4);
#pragma unroll
                    for (int k = 0; k < STEP; k += 16) save_run_f32(part, block, k, lane, v + k);
                }
                continue;
            }
            if (live) {
#pragma unroll
                for (int k = 0; k < STEP; k += 16) dense_pair_run<MODE, ACT, HALF, FLAGS>(p, v + k, u, has_res, panel, (c & 31) + k, col + (c & 31) + k, block);
            }
            if (!last) continue;
            ++used;
            if (out_tma) {
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) {
                    if (live) tma_store_2d(my, panel, col, row0);
                    bulk_commit();
                }
            } else if (live) {
                __syncwarp();
#pragma unroll 8
                for (int r = 0; r < 32; ++r)
                    if (row0 + r < p.T && col + lane < p.F)
                        p.out0[(long long)(row0 + r) * p.ld_out + col + lane] =
                            *reinterpret_cast<const unsigned short *>(panel + sw64_offset(r, lane >> 3) + (lane & 7) * 2);
                __syncwarp();
            }
            if (res_tma && lane == 0 && (used > 1 || panels == 1)) {  // the next panel's residual, once the store before this one has read its buffer
                bulk_wait_read<1>();
                fence_proxy_async();
                if (i + 1 < panels) fetch_residual(t, i + 1, b ^ 1);
                else if (next.valid()) fetch_residual(next, 0, b ^ 1);
            }
            __syncwarp();
        }
        t = next;
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
}

template <int MODE, int HALF, int FLAGS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(DP_THREADS, 1)
    dense_pair_kernel(const __grid_constant__ CUtensorMap ma0, const __grid_constant__ CUtensorMap ma1, const __grid_constant__ CUtensorMap mb0,
                      const __grid_constant__ CUtensorMap mb1, const __grid_constant__ CUtensorMap my, const __grid_constant__ CUtensorMap mr,
                      const __grid_constant__ DensePairParams p) {
    extern __shared__ __align__(1024) uint8_t dp_raw[];
    DensePairSmem &sm = *reinterpret_cast<DensePairSmem *>(dp_raw);
    if (smem_u32(dp_raw) & 1023) {  // the swizzled tiles need the alignment that the declaration asks for
        if (threadIdx.x == 0) atomicExch(&g_device_status, (int)PAI_ERR_MISALIGNED);
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    DensePairTiles t(p, (int)blockIdx.x >> 1, (int)gridDim.x >> 1);
    const int f_width = MODE == DP_GATED ? p.bn / 2 : p.bn;
    const int b_rows = p.bn / 2;  // rows of B this CTA stages

    if (warp == 2) asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512) : "memory");
    if (threadIdx.x == 0) {
        for (int i = 0; i < DP_STAGES; ++i) {
            mbar_init(&sm.full[i], 1);
            mbar_init(&sm.free[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.acc_full[i], 1);
            mbar_init(&sm.acc_free[i], 2 * DP_EPI_WARPS);
            
        }
        for (int w = 0; w < 2 * DP_EPI_WARPS; ++w) mbar_init(&sm.res_full[0][0] + w, 1);
        sm.abort_flag = 0;
        mbar_fence_init();
    }
    tc_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();  // both CTAs' barriers are ready
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    pdl_trigger();
    pdl_wait();

    // (The loops of warps 0 and 1 are run by the whole warp, one elected thread issuing: control flow and descriptors stay warp-uniform, which keeps
    // the instructions between two products few.  Run by one thread alone they took 620 cycles per reduction block, and 1200 beside a busy
    // epilogue, where the products themselves take 512.)
    if (warp == 0) {
        const bool leader = elect_one();
        int slot = 0;
        uint32_t phase = 0;
        bool ok = true;
        const uint32_t bytes = 2 * (16384 + (uint32_t)b_rows * 128), full0 = map_to_rank(smem_u32(&sm.full[0]), 0);
        for (; t.valid() && ok; t.next(p)) {
            const int ta = t.t * 256 + (int)rank * 128, fb = t.f * f_width + (MODE == DP_GATED ? 0 : (int)rank * b_rows), group = t.group(p);
            int k0, k1;
            t.range(p, k0, k1);
            for (int kb = k0; kb < k1; ++kb) {
                if (!mbar_wait_abortable(&sm.free[slot], phase ^ 1, &sm.abort_flag)) {
                    ok = false;
                    break;
                }
                if (leader) {
                    uint8_t *a = sm.stage[slot], *b = a + 16384;
                    if (rank == 0) mbar_expect_tx(&sm.full[slot], bytes);
                    const uint32_t bar = full0 + slot * 8;
                    const bool second = kb >= p.kb_seg;
                    const int r = (second ? kb - p.kb_seg : kb) * DP_BK;
                    const CUtensorMap *mA = (second || group) ? &ma1 : &ma0;
                    const CUtensorMap *mB = (second || (MODE == DP_GATED && rank)) ? &mb1 : &mb0;
                    if (p.a_mn) {
                        tma_load_2d_pair(a, mA, ta, r, bar);
                        tma_load_2d_pair(a + 8192, mA, ta + 64, r, bar);
                    } else {
                        tma_load_2d_pair(a, mA, r, ta, bar);
                    }
                    if (p.b_mn) {
                        for (int i = 0; i < b_rows; i += 64) tma_load_2d_pair(b + i * 128, mB, fb + i, r, bar);
                    } else {
                        tma_load_2d_pair(b, mB, r, fb, bar);
                    }
                }
                __syncwarp();
                if (++slot == DP_STAGES) slot = 0, phase ^= 1;
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const bool leader = elect_one();
            const uint32_t a_step = (p.a_mn ? 2048 : 32) >> 4, b_step = (p.b_mn ? 2048 : 32) >> 4;
            const uint64_t ad0 = umma_desc_sw128(smem_u32(sm.stage[0]), p.a_mn ? 8192 : 16, 1024);
            const uint64_t bd0 = umma_desc_sw128(smem_u32(sm.stage[0]) + 16384, p.b_mn ? 8192 : 16, 1024);
            int slot = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int n = 0; t.valid() && ok; t.next(p), ++n) {
                const int acc = n & 1;
                int k0, k1;
                t.range(p, k0, k1);
                if (!mbar_wait_abortable(&sm.acc_free[acc], ((n >> 1) & 1) ^ 1, &sm.abort_flag)) break;
                tc_fence_after();
                for (int kb = k0; kb < k1; ++kb) {
                    if (!mbar_wait_abortable(&sm.full[slot], phase, &sm.abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    if (leader) {
                        const uint64_t ad = ad0 + (uint64_t)(slot * (DP_STAGE_BYTES >> 4)), bd = bd0 + (uint64_t)(slot * (DP_STAGE_BYTES >> 4));
#pragma unroll
                        for (int k = 0; k < 4; ++k) umma_ss_pair(tmem + acc * 256, ad + k * a_step, bd + k * b_step, p.idesc, kb > k0 || k > 0);
                        umma_commit_pair(&sm.free[slot]);
                    }
                    __syncwarp();
                    if (++slot == DP_STAGES) slot = 0, phase ^= 1;
                }
                if (ok && leader) umma_commit_pair(&sm.acc_full[acc]);
                __syncwarp();
            }
        }
    } else if (warp == 3) {
        if (MODE != DP_GATED) dense_colsum<HALF>(p.colsum, (int)blockIdx.x, (int)gridDim.x);
    } else if (warp >= 4) {
        if (MODE == DP_PARTIAL) {
            dense_pair_epilogue<MODE, ACT_NONE, HALF, FLAGS>(p, sm, &my, &mr, tmem, rank, t);
        } else {
            switch (p.act) {
                case ACT_GELU: dense_pair_epilogue<MODE, ACT_GELU, HALF, FLAGS>(p, sm, &my, &mr, tmem, rank, t); break;
                case ACT_SILU: dense_pair_epilogue<MODE, ACT_SILU, HALF, FLAGS>(p, sm, &my, &mr, tmem, rank, t); break;
                case ACT_RELU: dense_pair_epilogue<MODE, ACT_RELU, HALF, FLAGS>(p, sm, &my, &mr, tmem, rank, t); break;
                case ACT_SIGMOID: dense_pair_epilogue<MODE, ACT_SIGMOID, HALF, FLAGS>(p, sm, &my, &mr, tmem, rank, t); break;
                default: dense_pair_epilogue<MODE, ACT_NONE, HALF, FLAGS>(p, sm, &my, &mr, tmem, rank, t);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();  // neither CTA leaves (nor frees tensor memory) while the other's products or arrivals may still touch it
    if (warp == 2) {
        tc_fence_after();
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// out[group][t, f] = sum over splits of the partial tiles, in order of the splits; a CTA per block of 32 x 32, a warp per four rows of it
__global__ void __launch_bounds__(256) dense_reduce_kernel(const float *__restrict__ part, unsigned short *out0, unsigned short *out1, int T, int F,
                                                           long long ld_out, int groups, int splits, int half) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, col_blocks = (F + 31) >> 5;
    const size_t matrix = saved_bytes_f32(T, F) / 4, b = blockIdx.x;
    const int group = blockIdx.y, r = (threadIdx.x >> 5) * 4 + (lane >> 3);
    unsigned short *out = group ? out1 : out0;
    const int t = (int)(b / col_blocks) * 32 + r, f = (int)(b % col_blocks) * 32 + (lane & 7) * 4;
    const float *src = part + group * matrix + b * 1024 + (lane & 7) * 128 + r * 4;
    float4 s = *reinterpret_cast<const float4 *>(src);
#pragma unroll 8
    for (int i = 1; i < splits; ++i) {
        const float4 v = *reinterpret_cast<const float4 *>(src + (size_t)i * groups * matrix);
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    if (t >= T) return;
    unsigned short *o = out + (long long)t * ld_out + f;
    if ((ld_out & 3) == 0 && ((uintptr_t)out & 7) == 0 && f + 4 <= F) {
        *reinterpret_cast<uint2 *>(o) = make_uint2(pack_bits16(s.x, s.y, half), pack_bits16(s.z, s.w, half));
    } else {
        const float e[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (f + i < F) o[i] = to_bits16(e[i], half);
    }
}

}  // namespace pai
