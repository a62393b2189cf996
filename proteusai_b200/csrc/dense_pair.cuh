// dense_pair_kernel: the products of the feed-forward block at sizes that fill the GPU.  out[t, f] = epilogue( sum_r A[t, r] B[f, r] ),
// one output tile of 256 t x bn f per CTA PAIR: tcgen05.mma.cta_group::2 (M = 256), each CTA of the pair staging its own 128 rows of A and
// half of B, so that a 64-wide reduction block costs each SM 32 KB from L2 per 512 tensor cycles at bn = 256 (64 bytes a cycle; single-CTA tiles of
// 128 x 128 need twice that and were bound by it).  Persistent: the pairs walk the tiles, the accumulator in tensor memory is doubled, and the
// epilogue of one tile runs under the products of the next.
//
// An accumulator lane is an output ROW here (the operands of dense_tile.cuh swapped): a thread of the epilogue holds runs of 32 columns, packs
// them to 16-byte words, and the tile leaves through shared memory by TMA stores (64 columns x 32 rows per warp and step).
//     forward  t = token,           f = output feature, r = input feature:  A = x  (K-major),  B = W (K-major)
//     gated    the same with B = 128 rows of Wg (staged by the pair's first CTA) and 128 of Wu (by its second): columns [0, 128) of the
//              accumulator are g, [128, 256) are u
//     dx       t = token,           f = input feature,  r = output feature: A = dz (K-major),  B = W (MN-major); gated: two pairs in sequence
//     dW       t = output feature,  f = input feature,  r = token:          A = dz (MN-major), B = x (MN-major); the long reduction split
//              over pairs that leave fp32 tiles in the workspace, added in order by dense_reduce_kernel
//
// Warps: 0 TMA loads, 1 MMAs (first CTA of the pair), 2 tensor memory, 4..11 epilogue (two per quarter of the lanes, half the columns each).
#pragma once
#include "dense_tile.cuh"

namespace pai {

constexpr int DP_THREADS = 384;
constexpr int DP_STAGES = 5;
constexpr int DP_STAGE_BYTES = 32768;  // A 128 x 128 bytes, B up to 128 x 128 bytes
constexpr int DP_EPI_WARPS = 8;

struct DensePairSmem {
    uint8_t stage[DP_STAGES][DP_STAGE_BYTES];
    uint8_t panel[DP_EPI_WARPS][2][4096];  // per epilogue warp: 32 rows x 128 bytes, 128-byte swizzle; output (and residual) staging
    float bias[2][256];
    uint64_t full[DP_STAGES], free[DP_STAGES], acc_full[2], acc_free[2];
    uint64_t res_full[DP_EPI_WARPS][2];
    uint32_t tmem;
    int abort_flag;
};

enum { DP_LINEAR = 0, DP_GATED = 1, DP_PARTIAL = 2 };

struct DensePairParams {
    unsigned short *out0;
    const unsigned short *residual;
    const void *bias0, *bias1;
    uint8_t *save0, *save1;          // saved pre-activations of g / z and u, or NULL
    float *part;                     // DP_PARTIAL: fp32 tiles, [split][group] matrices in the layout of saved_index_f32
    long long ld_out, ld_res, save_scale_off;
    int T, F, bn;                    // bn: accumulator columns of a tile (gated: bn / 2 of each)
    int t_tiles, f_tiles, groups, splits;
    int kb_seg, kb_total;
    int a_mn, b_mn, act, half, bias_fp32;
    int tma_out, tma_res, save_f32;
    uint32_t idesc;
};

// ---- CTA-pair forms of the helpers in tc.cuh --------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
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
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// ---- epilogue -------------------------------------------------------------------------------------------------------
// v[i] (32 columns of this thread's row) to the block; NaN and infinities keep their kind
__device__ __forceinline__ void save_run_f16(uint8_t *values, uint8_t *exps, size_t block, int row, const float (&v)[32]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) m = fmaxf(m, fabsf(v[i]));
    int e = (int)(__float_as_uint(m) >> 23) - 127 - 14;  // 2^e 2^14 <= m < 2^e 2^15
    if (m == 0.f || m > 3.4e38f) e = 0;
    e = e < -112 ? -112 : e;  // (2^-e stays finite; what is smaller than 2^-98 loses bits)
    const float s = __uint_as_float((uint32_t)(127 - e) << 23);
    uint4 *dst = reinterpret_cast<uint4 *>(values + block * 2048);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_bits16(v[q * 8 + 2 * i] * s, v[q * 8 + 2 * i + 1] * s, 1);
        dst[q * 32 + row] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    exps[block * 32 + row] = (uint8_t)(signed char)e;
}
__device__ __forceinline__ void save_run_f32(float *values, size_t block, int row, const float (&v)[32]) {
    float4 *dst = reinterpret_cast<float4 *>(values + block * 1024);
#pragma unroll
    for (int q = 0; q < 8; ++q) dst[q * 32 + row] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
}

__device__ __forceinline__ void load_run(uint32_t taddr, float (&v)[32]) {
    uint32_t u[32];
    tmem_ld32(taddr, u);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(u[i]);
}
__device__ __forceinline__ void add_bias_run(float (&v)[32], const float *bias) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float4 b = reinterpret_cast<const float4 *>(bias)[i];
        v[4 * i] += b.x, v[4 * i + 1] += b.y, v[4 * i + 2] += b.z, v[4 * i + 3] += b.w;
    }
}

// One 64-column panel of the tile for one warp: accumulators at `acc` (and `acc2`), output columns c0 .. c0 + 63 of rows row0 .. row0 + 31.
template <int MODE, int ACT>
__device__ __forceinline__ void dense_pair_panel(const DensePairParams &p, const CUtensorMap *my, uint8_t *panel, uint64_t *res_bar, uint32_t res_phase,
                                                 int *abort_flag, const float *bias, const float *bias2, uint32_t acc, uint32_t acc2, int c0, int row0,
                                                 float *part) {
    const int lane = threadIdx.x & 31;
    const int col_blocks = (p.F + 31) >> 5;
    const bool rows_in = row0 < p.T;  // (warp-uniform; saved blocks and partial tiles exist for whole blocks of 32 rows)
    if (MODE == DP_LINEAR && p.residual) {
        if (p.tma_res) {
            if (rows_in && c0 < p.F) mbar_wait_abortable(res_bar, res_phase, abort_flag);
        } else {
            for (int r = 0; r < 32; ++r) {  // any alignment: a row at a time, two columns per lane
                const int t = row0 + r;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int c = h * 32 + lane;
                    const unsigned short v = t < p.T && c0 + c < p.F ? p.residual[(long long)t * p.ld_res + c0 + c] : (unsigned short)0;
                    *reinterpret_cast<unsigned short *>(panel + sw128_offset(r, c >> 3) + (c & 7) * 2) = v;
                }
            }
            __syncwarp();
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int c = c0 + h * 32;
        float v[32];
        load_run(acc + h * 32, v);
        const bool live = rows_in && c < p.F;
        if (MODE == DP_PARTIAL) {
            if (live) save_run_f32(part, saved_block(row0, c, col_blocks), lane, v);
            continue;
        }
        if (p.bias0) add_bias_run(v, bias + h * 32);
        float u[32];
        if (MODE == DP_GATED) {
            load_run(acc2 + h * 32, u);
            if (p.bias1) add_bias_run(u, bias2 + h * 32);
        }
        if (p.save0 && live) {
            const size_t block = saved_block(row0, c, col_blocks);
            if (p.save_f32) {
                save_run_f32(reinterpret_cast<float *>(p.save0), block, lane, v);
                if (MODE == DP_GATED) save_run_f32(reinterpret_cast<float *>(p.save1), block, lane, u);
            } else {
                save_run_f16(p.save0, p.save0 + p.save_scale_off, block, lane, v);
                if (MODE == DP_GATED) save_run_f16(p.save1, p.save1 + p.save_scale_off, block, lane, u);
            }
        }
#pragma unroll
        for (int i = 0; i < 32; i += 2) act_pair<ACT>(v[i], v[i + 1]);
        if (MODE == DP_GATED) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] *= u[i];
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint4 *at = reinterpret_cast<uint4 *>(panel + sw128_offset(lane, h * 4 + q));
            if (MODE == DP_LINEAR && p.residual) {
                const uint4 r = *at;
                const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float lo, hi;
                    unpack_bits16(w[i], p.half, lo, hi);
                    v[q * 8 + 2 * i] += lo, v[q * 8 + 2 * i + 1] += hi;
                }
            }
            *at = make_uint4(pack_bits16(v[q * 8], v[q * 8 + 1], p.half), pack_bits16(v[q * 8 + 2], v[q * 8 + 3], p.half),
                             pack_bits16(v[q * 8 + 4], v[q * 8 + 5], p.half), pack_bits16(v[q * 8 + 6], v[q * 8 + 7], p.half));
        }
    }
    if (MODE == DP_PARTIAL) return;
    if (p.tma_out) {
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
            if (rows_in && c0 < p.F) tma_store_2d(my, panel, c0, row0);
            bulk_commit();
        }
    } else {
        __syncwarp();
        for (int r = 0; r < 32; ++r) {
            const int t = row0 + r;
            if (t >= p.T) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int c = h * 32 + lane;
                if (c0 + c < p.F)
                    p.out0[(long long)t * p.ld_out + c0 + c] = *reinterpret_cast<const unsigned short *>(panel + sw128_offset(r, c >> 3) + (c & 7) * 2);
            }
        }
        __syncwarp();
    }
}

struct DensePairTile {
    int t0, f0, group, split, k0, k1;
};
__device__ __forceinline__ DensePairTile dense_pair_tile(const DensePairParams &p, int item, int f_width) {
    DensePairTile t;
    t.f0 = (item % p.f_tiles) * f_width;
    item /= p.f_tiles;
    t.t0 = (item % p.t_tiles) * 256;
    item /= p.t_tiles;
    t.group = item % p.groups;
    t.split = item / p.groups;
    t.k0 = (int)((long long)p.kb_total * t.split / p.splits);
    t.k1 = (int)((long long)p.kb_total * (t.split + 1) / p.splits);
    return t;
}

template <int MODE, int ACT>
__device__ __forceinline__ void dense_pair_epilogue(const DensePairParams &p, DensePairSmem &sm, const CUtensorMap *my, const CUtensorMap *mr,
                                                    uint32_t tmem, uint32_t rank, int items, int pairs) {
    const int warp = (threadIdx.x >> 5) - 4, lane = threadIdx.x & 31, q = warp & 3, half = warp >> 2;
    const int f_width = MODE == DP_GATED ? p.bn / 2 : p.bn;
    const int panels = f_width / 128;  // 64-column panels of this warp: half the tile's columns
    const uint32_t acc_free0 = map_to_rank(smem_u32(&sm.acc_free[0]), 0), acc_free1 = map_to_rank(smem_u32(&sm.acc_free[1]), 0);
    int n = 0, used = 0;     // tiles done, panels done (the two staging buffers alternate)
    uint32_t res_phase = 0;  // bit i: phase of res_full[i]
    for (int item = blockIdx.x >> 1; item < items; item += pairs, ++n) {
        const DensePairTile t = dense_pair_tile(p, item, f_width);
        const int row0 = t.t0 + (int)rank * 128 + q * 32, col0 = t.f0 + half * panels * 64;
        const int a = n & 1;
        if (MODE != DP_PARTIAL && (p.bias0 || (MODE == DP_GATED && p.bias1))) {
            const int i = threadIdx.x - 128;  // 0 .. 255: column of the accumulator
            const void *b = MODE == DP_GATED && i >= f_width ? p.bias1 : p.bias0;
            const int c = t.f0 + (MODE == DP_GATED && i >= f_width ? i - f_width : i);
            sm.bias[a][i] = b && c < p.F && i < p.bn ? load_bias(b, c, p.bias_fp32, p.half) : 0.f;
            asm volatile("bar.sync 1, 256;" ::: "memory");
        }
        if (MODE == DP_LINEAR && p.residual && p.tma_res && lane == 0) {
            bulk_wait_read<0>();  // the panels' last stores have been read out of shared memory
            fence_proxy_async();
            for (int i = 0; i < panels; ++i)
                if (row0 < p.T && col0 + i * 64 < p.F) {
                    const int b = (used + i) & 1;
                    mbar_expect_tx(&sm.res_full[warp][b], 4096);
                    tma_load_2d(sm.panel[warp][b], mr, col0 + i * 64, row0, &sm.res_full[warp][b]);
                }
        }
        __syncwarp();
        const bool ok = mbar_wait_abortable(&sm.acc_full[a], (n >> 1) & 1, &sm.abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t acc = tmem + a * 256 + ((uint32_t)(q * 32) << 16) + half * panels * 64;
        float *part = MODE == DP_PARTIAL ? p.part + (size_t)(t.split * p.groups + t.group) * (saved_bytes_f32(p.T, p.F) / 4) : nullptr;
        for (int i = 0; i < panels; ++i, ++used) {
            const int b = used & 1;
            if (MODE != DP_PARTIAL && !(MODE == DP_LINEAR && p.residual && p.tma_res)) {
                if (lane == 0) bulk_wait_read<1>();  // this buffer's previous store has been read
                __syncwarp();
            }
            dense_pair_panel<MODE, ACT>(p, my, sm.panel[warp][b], &sm.res_full[warp][b], (res_phase >> b) & 1, &sm.abort_flag,
                                        &sm.bias[a][half * panels * 64 + i * 64], &sm.bias[a][(MODE == DP_GATED ? f_width : 0) + half * panels * 64 + i * 64],
                                        acc + i * 64, acc + f_width + i * 64, col0 + i * 64, row0, part);
            if (MODE == DP_LINEAR && p.residual && p.tma_res && row0 < p.T && col0 + i * 64 < p.F) res_phase ^= 1u << b;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(a ? acc_free1 : acc_free0);
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
}

template <int MODE>
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
    const int pairs = gridDim.x >> 1;
    const int items = p.f_tiles * p.t_tiles * p.groups * p.splits;
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
            for (int w = 0; w < DP_EPI_WARPS; ++w) mbar_init(&sm.res_full[w][i], 1);
        }
        sm.abort_flag = 0;
        mbar_fence_init();
    }
    tc_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();  // both CTAs' barriers are ready
    tc_fence_after();
    const uint32_t tmem = sm.tmem;

    if (warp == 0) {
        if (lane == 0) {
            int slot = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int item = blockIdx.x >> 1; item < items && ok; item += pairs) {
                const DensePairTile t = dense_pair_tile(p, item, f_width);
                const int ta = t.t0 + (int)rank * 128;
                const int fb = MODE == DP_GATED ? t.f0 : t.f0 + (int)rank * b_rows;
                for (int kb = t.k0; kb < t.k1; ++kb) {
                    if (!mbar_wait_abortable(&sm.free[slot], phase ^ 1, &sm.abort_flag)) {
                        ok = false;
                        break;
                    }
                    uint8_t *a = sm.stage[slot], *b = a + 16384;
                    if (rank == 0) mbar_expect_tx(&sm.full[slot], 2 * (16384 + (uint32_t)b_rows * 128));
                    const uint32_t bar = map_to_rank(smem_u32(&sm.full[slot]), 0);
                    const bool second = kb >= p.kb_seg;
                    const int r = (second ? kb - p.kb_seg : kb) * DT_BK;
                    const CUtensorMap *mA = (second || t.group) ? &ma1 : &ma0;
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
                    if (++slot == DP_STAGES) slot = 0, phase ^= 1;
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const uint32_t a_step = (p.a_mn ? 2048 : 32) >> 4, b_step = (p.b_mn ? 2048 : 32) >> 4;
            const uint64_t ad0 = umma_desc_sw128(smem_u32(sm.stage[0]), p.a_mn ? 8192 : 16, 1024);
            const uint64_t bd0 = umma_desc_sw128(smem_u32(sm.stage[0]) + 16384, p.b_mn ? 8192 : 16, 1024);
            int slot = 0, n = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int item = blockIdx.x >> 1; item < items && ok; item += pairs, ++n) {
                const DensePairTile t = dense_pair_tile(p, item, f_width);
                const int acc = n & 1;
                if (!mbar_wait_abortable(&sm.acc_free[acc], ((n >> 1) & 1) ^ 1, &sm.abort_flag)) break;
                tc_fence_after();
                for (int kb = t.k0; kb < t.k1; ++kb) {
                    if (!mbar_wait_abortable(&sm.full[slot], phase, &sm.abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t ad = ad0 + (uint64_t)slot * (DP_STAGE_BYTES >> 4), bd = bd0 + (uint64_t)slot * (DP_STAGE_BYTES >> 4);
#pragma unroll
                    for (int k = 0; k < 4; ++k) umma_ss_pair(tmem + acc * 256, ad + k * a_step, bd + k * b_step, p.idesc, kb > t.k0 || k > 0);
                    umma_commit_pair(&sm.free[slot]);
                    if (++slot == DP_STAGES) slot = 0, phase ^= 1;
                }
                if (ok) umma_commit_pair(&sm.acc_full[acc]);
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        if (MODE == DP_PARTIAL) {
            dense_pair_epilogue<MODE, ACT_NONE>(p, sm, &my, &mr, tmem, rank, items, pairs);
        } else {
            switch (p.act) {
                case ACT_GELU: dense_pair_epilogue<MODE, ACT_GELU>(p, sm, &my, &mr, tmem, rank, items, pairs); break;
                case ACT_SILU: dense_pair_epilogue<MODE, ACT_SILU>(p, sm, &my, &mr, tmem, rank, items, pairs); break;
                case ACT_RELU: dense_pair_epilogue<MODE, ACT_RELU>(p, sm, &my, &mr, tmem, rank, items, pairs); break;
                case ACT_SIGMOID: dense_pair_epilogue<MODE, ACT_SIGMOID>(p, sm, &my, &mr, tmem, rank, items, pairs); break;
                default: dense_pair_epilogue<MODE, ACT_NONE>(p, sm, &my, &mr, tmem, rank, items, pairs);
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

// out[group][t, f] = sum over splits of the partial tiles, in order of the splits; one warp per block of 32 x 32
__global__ void __launch_bounds__(256) dense_reduce_kernel(const float *__restrict__ part, unsigned short *out0, unsigned short *out1, int T, int F,
                                                           long long ld_out, int groups, int splits, int half) {
    const int lane = threadIdx.x & 31, col_blocks = (F + 31) >> 5;
    const size_t matrix = saved_bytes_f32(T, F) / 4, blocks = matrix / 1024;
    const size_t b = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (b >= blocks) return;
    const int group = blockIdx.y;
    unsigned short *out = group ? out1 : out0;
    const int t0 = (int)(b / col_blocks) * 32, f = (int)(b % col_blocks) * 32 + (lane & 7) * 4;
    const bool vec = (ld_out & 3) == 0 && ((uintptr_t)out & 7) == 0;
#pragma unroll
    for (int g = 0; g < 8; ++g) {
        const int r = g * 4 + (lane >> 3);
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = 0; i < splits; ++i) {
            const float4 v = *reinterpret_cast<const float4 *>(part + (size_t)(i * groups + group) * matrix + b * 1024 + (lane & 7) * 128 + r * 4);
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
        if (t0 + r < T) {
            unsigned short *o = out + (long long)(t0 + r) * ld_out + f;
            if (vec && f + 4 <= F) {
                *reinterpret_cast<uint2 *>(o) = make_uint2(pack_bits16(s.x, s.y, half), pack_bits16(s.z, s.w, half));
            } else {
                const float e[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (f + i < F) o[i] = to_bits16(e[i], half);
            }
        }
    }
}

}  // namespace pai
