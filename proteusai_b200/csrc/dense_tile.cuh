// dense_tile_kernel: out[t, f] = epilogue( sum_r A[f, r] B[t, r] ) on the tensor cores, one output tile of 128 f x tn t per CTA, the
// reduction split over a cluster where there are too few tiles to fill the GPU.
//
// The contiguous axis of the output (f) is the M axis of the MMA: a few tokens cost an MMA of N = 16 rather than 128 rows of which a few are
// wanted.  The same kernel runs every product of the two operators:
//     forward   f = output feature, t = token,           r = input feature:   A = W        (K-major),  B = x  (K-major)
//     dx        f = input feature,  t = token,           r = output feature:  A = W        (MN-major), B = dz (K-major)
//     dW        f = input feature,  t = output feature,  r = token:           A = x        (MN-major), B = dz (MN-major)
// Gated forward: two A operands (Wg, Wu) against one B into two accumulators (DUAL).  Gated dx: two pairs of operands in sequence into one
// accumulator (kb_seg).  Gated dW: two output groups (the second with its own B and output).
//
// Split reduction: the CTAs of a cluster each take a run of the reduction blocks and send their partial rows to the CTA that finishes
// them (tn / splits rows each) by bulk copies into its shared memory; that CTA adds the partials of all ranks in rank order: one launch, no
// workspace, no atomics, the same bits every time.  The cluster barriers around the copies are arrived at long before they are waited for.
//
// Tensor memory is given back before a CTA waits for the others' partials: one that waits never holds columns that another may need.
#pragma once
#include "dense_ops.cuh"
#include "tc.cuh"

namespace pai {

constexpr int DT_THREADS = 256;
constexpr int DT_FT = 128;        // output columns (MMA rows) per tile
constexpr int DT_BK = 128;        // reduction block: two swizzle rows of 64.  (With 64 the wait, commit and loop around four MMAs cost as much as they.)
constexpr int DT_MAX_STAGES = 8;

struct DenseTileParams {
    void *out0, *out1;              // 16-bit outputs of the groups
    const void *bias0, *bias1;      // [F] of the accumulators (DUAL: both), or NULL
    const unsigned short *residual; // [T, F], or NULL
    float *save0, *save1;           // saved pre-activations (saved_index_f32), or NULL
    long long ld_out, ld_res;
    int F, T;
    int splits, split_log, tn, stages;  // splits = 1 << split_log; grid: x = t tile * splits + rank, y = f tile, z = group
    int kb_seg, kb_total;           // reduction blocks of the first operand pair, of both
    int tail;                       // the last block of a pair has 64 columns at most
    int a_mn, b_mn;                 // operands stored with the reduction as their slow axis
    int act, bias_fp32;
    uint32_t idesc;
    DenseColsum colsum;             // bias gradients to finish beside the product
};

__device__ __forceinline__ void tma_load_2d(void *dst_smem, const CUtensorMap *map, int c0, int c1, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst_smem)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
        : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// one thread of a converged warp
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// bulk copy from this CTA's shared memory into that of a CTA of the cluster; its bytes count on that CTA's barrier
__device__ __forceinline__ void bulk_s2s(uint32_t dst, const void *src_smem, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "r"(smem_u32(src_smem)),
                 "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ float load_bias(const void *b, int i, int fp32, int half) {
    return fp32 ? reinterpret_cast<const float *>(b)[i] : from_bits16(reinterpret_cast<const unsigned short *>(b)[i], half);
}

// Rows [0, n) of `src` (row r at src + r DT_FT, DUAL: the second accumulator `second` floats behind; `splits` partial tiles `part` floats apart,
// added in order) are rows first + r of the output.  A warp takes a row at a time, a lane four columns from f: these calls are short chains of
// instructions on few warps, and a column per thread made this the longest part of a small product.
template <bool DUAL, int HALF>
__device__ __forceinline__ void dense_finish(const DenseTileParams &p, const float *src, int splits, int part, int second, int n, int first, int f,
                                             const float (&b0)[4], const float (&b1)[4], int group) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (f >= p.F) return;
    unsigned short *out = reinterpret_cast<unsigned short *>(group ? p.out1 : p.out0);
    const int col_blocks = (p.F + 31) >> 5, nf = p.F - f;
    const bool vec_out = nf >= 4 && (p.ld_out & 3) == 0 && ((uintptr_t)out & 7) == 0;
    const bool vec_res = nf >= 4 && (p.ld_res & 3) == 0 && ((uintptr_t)p.residual & 7) == 0;
#pragma unroll 1
    for (int r = warp; r < n; r += DT_THREADS / 32) {
        const long long t = first + r;
        unsigned short res[4] = {0, 0, 0, 0};
        if (p.residual) {
            const unsigned short *at = p.residual + t * p.ld_res + f;
            if (vec_res) {
                const uint2 w = *reinterpret_cast<const uint2 *>(at);
                res[0] = (unsigned short)w.x, res[1] = (unsigned short)(w.x >> 16), res[2] = (unsigned short)w.y, res[3] = (unsigned short)(w.y >> 16);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i < nf) res[i] = at[i];
            }
        }
        float v[4], u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = b0[i], u[i] = b1[i];
        const float *at = src + r * DT_FT + lane * 4;
        float4 x = *reinterpret_cast<const float4 *>(at), y = make_float4(0.f, 0.f, 0.f, 0.f);
        if (DUAL) y = *reinterpret_cast<const float4 *>(at + second);
        for (int s = 1; s < splits; ++s) {
            at += part;
            const float4 a = *reinterpret_cast<const float4 *>(at);
            x.x += a.x, x.y += a.y, x.z += a.z, x.w += a.w;
            if (DUAL) {
                const float4 b = *reinterpret_cast<const float4 *>(at + second);
                y.x += b.x, y.y += b.y, y.z += b.z, y.w += b.w;
            }
        }
        v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
        if (DUAL) u[0] += y.x, u[1] += y.y, u[2] += y.z, u[3] += y.w;
        if (p.save0) {  // (the buffer's blocks reach past F)
            const size_t to = saved_index_f32(t, f, col_blocks);
            *reinterpret_cast<float4 *>(p.save0 + to) = make_float4(v[0], v[1], v[2], v[3]);
            if (DUAL) *reinterpret_cast<float4 *>(p.save1 + to) = make_float4(u[0], u[1], u[2], u[3]);
        }
        switch (p.act) {
            case ACT_GELU: act_pair<ACT_GELU>(v[0], v[1]), act_pair<ACT_GELU>(v[2], v[3]); break;
            case ACT_SILU: act_pair<ACT_SILU>(v[0], v[1]), act_pair<ACT_SILU>(v[2], v[3]); break;
            case ACT_RELU: act_pair<ACT_RELU>(v[0], v[1]), act_pair<ACT_RELU>(v[2], v[3]); break;
            case ACT_SIGMOID: act_pair<ACT_SIGMOID>(v[0], v[1]), act_pair<ACT_SIGMOID>(v[2], v[3]); break;
            default: break;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (DUAL) v[i] *= u[i];
            if (p.residual) v[i] += from_bits16(res[i], HALF);
        }
        unsigned short *o = out + t * p.ld_out + f;
        if (vec_out) {
            *reinterpret_cast<uint2 *>(o) = make_uint2(pack_bits16(v[0], v[1], HALF), pack_bits16(v[2], v[3], HALF));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < nf) o[i] = to_bits16(v[i], HALF);
        }
    }
}

template <bool DUAL, int HALF>
__global__ void __launch_bounds__(DT_THREADS, 2) dense_tile_kernel(const __grid_constant__ CUtensorMap ma0, const __grid_constant__ CUtensorMap ma1,
                                                                const __grid_constant__ CUtensorMap mb0, const __grid_constant__ CUtensorMap mb1,
                                                                const __grid_constant__ DenseTileParams p) {
    extern __shared__ uint8_t dt_raw[];
    __shared__ uint64_t bar_full[DT_MAX_STAGES], bar_free[DT_MAX_STAGES], bar_done, bar_red;
    __shared__ uint32_t tmem_base;
    __shared__ int abort_flag;
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(dt_raw) + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // (no divisions: the addresses of the first loads are what a small call waits for)
    const int rank = (int)blockIdx.x & (p.splits - 1), group = (int)blockIdx.z;
    const int f0 = (int)blockIdx.y * DT_FT, t0 = ((int)blockIdx.x >> p.split_log) * p.tn;
    const int k0 = (p.kb_total * rank) >> p.split_log, k1 = (p.kb_total * (rank + 1)) >> p.split_log;
    const int rows = p.tn >> p.split_log;  // rows of the tile that this CTA finishes
    constexpr int ACC = DUAL ? 2 : 1;
    // a stage: A (DUAL: both), B, each two K-major tiles of 64 columns or 64-wide panels of 128 steps of the reduction
    const uint32_t a_bytes = ACC * DT_FT * 256, b_bytes = (uint32_t)p.tn * 256, b_half = (uint32_t)p.tn * 128;
    const uint32_t stage_bytes = a_bytes + b_bytes;
    const uint32_t tile_bytes = (uint32_t)p.tn * ACC * DT_FT * 4;  // a whole partial tile, sent (over the stages) and received (behind them)
    float *red = reinterpret_cast<float *>(base + ((uint32_t)p.stages * stage_bytes > tile_bytes ? (uint32_t)p.stages * stage_bytes : tile_bytes));
    uint32_t cols = 32;
    while (cols < (uint32_t)p.tn * ACC) cols <<= 1;

    const int f = f0 + lane * 4;  // this thread's four output columns in the epilogue
    // (the loops of warps 0 and 1 are run by the whole warp, one elected thread issues: control flow and descriptors stay warp-uniform)
    const bool leader = warp < 2 && elect_one();
    auto load = [&](int kb, int slot) {
        uint8_t *a = base + (size_t)slot * stage_bytes, *b = a + a_bytes;
        mbar_expect_tx(&bar_full[slot], stage_bytes);
        const bool second = kb >= p.kb_seg;
        const int r = (second ? kb - p.kb_seg : kb) * DT_BK;
        const CUtensorMap *ma = second ? &ma1 : &ma0, *mb = (second || group) ? &mb1 : &mb0;
        if (p.a_mn) {
            tma_load_2d(a, ma, f0, r, &bar_full[slot]);
            tma_load_2d(a + 16384, ma, f0 + 64, r, &bar_full[slot]);
        } else {
            tma_load_2d(a, ma, r, f0, &bar_full[slot]);
            tma_load_2d(a + 16384, ma, r + 64, f0, &bar_full[slot]);
            if (DUAL) {
                tma_load_2d(a + 32768, &ma1, r, f0, &bar_full[slot]);
                tma_load_2d(a + 49152, &ma1, r + 64, f0, &bar_full[slot]);
            }
        }
        if (p.b_mn) {
            for (int i = 0; i < p.tn; i += 64) tma_load_2d(b + i * 256, mb, t0 + i, r, &bar_full[slot]);
        } else {
            tma_load_2d(b, mb, r, t0, &bar_full[slot]);
            tma_load_2d(b + b_half, mb, r + 64, t0, &bar_full[slot]);
        }
    };
    const int fresh = k1 - k0 < p.stages ? k1 - k0 : p.stages;  // loads that need no free slot; the first two are under way before the rest is set up
    const int ahead = fresh < 2 ? fresh : 2;
    if (warp == 0) {
        if (leader) {
            for (int i = 0; i < p.stages; ++i) {
                mbar_init(&bar_full[i], 1);
                mbar_init(&bar_free[i], 1);
            }
            mbar_init(&bar_done, 1);
            mbar_init(&bar_red, 1);
            abort_flag = 0;
            mbar_fence_init();
            if (p.splits > 1) {
                const int left = p.T - t0 - rank * rows;
                mbar_expect_tx(&bar_red, (uint32_t)(p.splits * ACC * (left < 0 ? 0 : left < rows ? left : rows) * DT_FT * 4));
            }
        }
        __syncwarp();
        pdl_wait();
        if (leader)
            for (int i = 0; i < ahead; ++i) load(k0 + i, i);
        __syncwarp();
    } else {
        pdl_wait();
    }
    if (p.splits > 1) cluster_arrive();  // (this CTA's barriers are ready)
    if (warp == 2) tmem_alloc(&tmem_base, cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base;
    pdl_trigger();

    if (warp == 0) {
        if (leader)
            for (int i = ahead; i < fresh; ++i) load(k0 + i, i);
        __syncwarp();
        int slot = fresh == p.stages ? 0 : fresh;
        uint32_t phase = fresh == p.stages ? 1 : 0;
        for (int kb = k0 + fresh; kb < k1; ++kb) {
            if (!mbar_wait_abortable(&bar_free[slot], phase ^ 1, &abort_flag)) break;
            if (leader) load(kb, slot);
            __syncwarp();
            if (++slot == p.stages) slot = 0, phase ^= 1;
        }
    } else if (warp == 1) {
        // K-major: rows of 128 bytes, 8-row groups 1024 apart, 16 elements of the reduction 32 bytes on, the next 64 in the next tile.
        // MN-major: 64-wide panels 16384 apart, 8 steps of the reduction 1024 apart, 16 of them 2048 on.
        const uint32_t a_step = (p.a_mn ? 2048 : 32) >> 4, b_step = (p.b_mn ? 2048 : 32) >> 4;
        const uint32_t a_next = (p.a_mn ? 8192 : 16384) >> 4, b_next = (p.b_mn ? 8192 : b_half) >> 4;
        const uint64_t ad0 = umma_desc_sw128(smem_u32(base), p.a_mn ? 16384 : 16, 1024);
        const uint64_t bd0 = umma_desc_sw128(smem_u32(base) + a_bytes, p.b_mn ? 16384 : 16, 1024);
        int slot = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int kb = k0; kb < k1; ++kb) {
            if (!mbar_wait_abortable(&bar_full[slot], phase, &abort_flag)) {
                ok = false;
                break;
            }
            tc_fence_after();
            if (leader) {
                const uint64_t ad = ad0 + (uint64_t)(slot * (stage_bytes >> 4)), bd = bd0 + (uint64_t)(slot * (stage_bytes >> 4));
                const bool half = p.tail && (kb + 1 == p.kb_seg || kb + 1 == p.kb_total);  // (its second 64 columns are zeros)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (h == 0 || !half) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint64_t ak = ad + h * a_next + k * a_step, bk = bd + h * b_next + k * b_step;
                            umma_ss(tmem, ak, bk, p.idesc, kb > k0 || h > 0 || k > 0);
                            if (DUAL) umma_ss(tmem + p.tn, ak + (32768 >> 4), bk, p.idesc, kb > k0 || h > 0 || k > 0);
                        }
                    }
                umma_commit(&bar_free[slot]);
            }
            __syncwarp();
            if (++slot == p.stages) slot = 0, phase ^= 1;
        }
        if (ok && leader) umma_commit(&bar_done);
    } else if (warp == 3) {
        dense_colsum<HALF>(p.colsum, (int)(blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z)), (int)(gridDim.x * gridDim.y * gridDim.z));
    }
    __syncwarp();
    float b0[4], b1[4];  // (on their way while the products run)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        b0[i] = p.bias0 && f + i < p.F ? load_bias(p.bias0, f + i, p.bias_fp32, HALF) : 0.f;
        b1[i] = DUAL && p.bias1 && f + i < p.F ? load_bias(p.bias1, f + i, p.bias_fp32, HALF) : 0.f;
    }
    bool ok = mbar_wait_abortable(&bar_done, 0, &abort_flag);
    tc_fence_after();
    float *mine = reinterpret_cast<float *>(base);  // over the stages, which have been read: this CTA's tile [accumulator][tn][128]
    if (ok) {
        const int q = warp & 3;
        for (int c = (warp >> 2) * 16; c < p.tn * ACC; c += 32) {
            const int tc = DUAL && c >= p.tn ? c - p.tn : c;
            if (t0 + tc >= p.T) continue;  // (warp-uniform)
            uint32_t v[16];
            tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + c, v);
            tmem_wait_ld();
            float *to = mine + c * DT_FT + q * 32 + lane;
#pragma unroll
            for (int j = 0; j < 16; ++j) to[j * DT_FT] = __uint_as_float(v[j]);
        }
    }
    if (p.splits > 1) fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        tmem_relinquish();
        tmem_dealloc(tmem, cols);
    }
    __syncwarp();
    const int first = t0 + rank * rows, left = p.T - first, n = left < rows ? left : rows;  // rows that are this CTA's to finish
    if (p.splits > 1) {
        cluster_wait();  // every CTA of the cluster has its barriers: it can be sent to
        if (warp == 0 && lane < p.splits && ok) {
            const int left_to = p.T - t0 - lane * rows, to = left_to < 0 ? 0 : left_to < rows ? left_to : rows;  // rows that rank `lane` finishes
            const uint32_t bar = map_to_rank(smem_u32(&bar_red), lane);
#pragma unroll
            for (int a = 0; a < ACC; ++a)
                if (to > 0)
                    bulk_s2s(map_to_rank(smem_u32(red + (rank * ACC + a) * rows * DT_FT), lane), mine + (a * p.tn + lane * rows) * DT_FT,
                             (uint32_t)to * DT_FT * 4, bar);
        }
        __syncwarp();
        ok = mbar_wait_abortable(&bar_red, 0, &abort_flag) && ok;
        cluster_arrive();
    }
    if (ok) {
        if (p.splits > 1) dense_finish<DUAL, HALF>(p, red, p.splits, ACC * rows * DT_FT, rows * DT_FT, n, first, f, b0, b1, group);
        else dense_finish<DUAL, HALF>(p, mine, 1, 0, p.tn * DT_FT, n, first, f, b0, b1, group);
    }
    __syncwarp();
    if (p.splits > 1) cluster_wait();  // what this CTA sent has been received
}

}  // namespace pai
