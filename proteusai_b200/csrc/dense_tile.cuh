// dense_tile_kernel: out[t, f] = epilogue( sum_r A[f, r] B[t, r] ) on the tensor cores, one output tile of 128 f x tn t per CTA, the
// reduction split over a cluster where there are too few tiles to fill the GPU.
//
// The contiguous axis of the output (f) is the M axis of the MMA, so an accumulator lane is an output column: the 32 lanes of a warp store
// 64 contiguous bytes of a row, a bias is one register per thread, and a single token costs an MMA of N = 16 rather than 128 rows of
// which one is wanted.  The same kernel runs every product of the two operators:
//     forward   f = output feature, t = token,           r = input feature:   A = W        (K-major),  B = x  (K-major)
//     dx        f = input feature,  t = token,           r = output feature:  A = W        (MN-major), B = dz (K-major)
//     dW        f = input feature,  t = output feature,  r = token:           A = x        (MN-major), B = dz (MN-major)
// Gated forward: two A operands (Wg, Wu) against one B into two accumulators (DUAL).  Gated dx: two pairs of operands in sequence into one
// accumulator (kb_seg).  Gated dW: two output groups (the second with its own B and output).
//
// Split reduction: the CTAs of a cluster each take a run of the 64-wide reduction blocks and send their partial rows to the CTA that finishes
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
constexpr int DT_BK = 64;         // reduction block: 128 bytes, one swizzle row
constexpr int DT_MAX_STAGES = 8;

struct DenseTileParams {
    void *out0, *out1;              // 16-bit outputs of the groups
    const void *bias0, *bias1;      // [F] of the accumulators (DUAL: both), or NULL
    const unsigned short *residual; // [T, F], or NULL
    float *save0, *save1;           // saved pre-activations (saved_index_f32), or NULL
    long long ld_out, ld_res;
    int F, T;
    int splits, split_log, tn, stages;  // splits = 1 << split_log; grid: x = t tile * splits + rank, y = f tile, z = group
    int kb_seg, kb_total;           // 64-wide reduction blocks of the first operand pair, of both
    int a_mn, b_mn;                 // operands stored with the reduction as their slow axis
    int act, bias_fp32;
    uint32_t idesc;
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

// One value of the output from its accumulator(s): column f (bias in b0, b1), row t.
template <bool DUAL, int ACT>
__device__ __forceinline__ float dense_finish(const DenseTileParams &p, float v0, float v1, float b0, float b1, int f, int t, int col_blocks) {
    v0 += b0;
    if (DUAL) v1 += b1;
    if (p.save0) {
        const size_t at = saved_index_f32(t, f, col_blocks);
        p.save0[at] = v0;
        if (DUAL) p.save1[at] = v1;
    }
    float dummy = 0.f;
    act_pair<ACT>(v0, dummy);
    return DUAL ? v0 * v1 : v0;
}

template <bool DUAL, int ACT, int HALF>
__device__ __forceinline__ void dense_epilogue(const DenseTileParams &p, uint32_t tmem, float *red, int f, float b0, float b1, int t0,
                                               int group, int rank) {
    const int tid = threadIdx.x, warp = tid >> 5;
    unsigned short *out = reinterpret_cast<unsigned short *>(group ? p.out1 : p.out0);
    const int col_blocks = (p.F + 31) >> 5;
    if (p.splits == 1) {
        const int q = warp & 3;
        const bool live = f < p.F;
        for (int c = (warp >> 2) * 16; c < p.tn; c += 32) {
            if (t0 + c >= p.T) break;  // (warp-uniform)
            uint32_t v[16], u[16];
            tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + c, v);
            if (DUAL) tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + p.tn + c, u);
            float r[16];
            const int nt = p.T - t0 - c;
            if (p.residual) {
#pragma unroll
                for (int j = 0; j < 16; ++j) r[j] = (live && j < nt) ? from_bits16(p.residual[(long long)(t0 + c + j) * p.ld_res + f], HALF) : 0.f;
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) r[j] = 0.f;
            }
            tmem_wait_ld();
            if (live) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (j < nt) {
                        const int t = t0 + c + j;
                        const float y = dense_finish<DUAL, ACT>(p, __uint_as_float(v[j]), DUAL ? __uint_as_float(u[j]) : 0.f, b0, b1, f, t, col_blocks);
                        out[(long long)t * p.ld_out + f] = to_bits16(y + r[j], HALF);
                    }
            }
            __syncwarp();
        }
        return;
    }
    // the ranks' partial rows [rank][accumulator][row][128 f]: this CTA's rows [rank, rank + 1) tn / splits of the tile
    const int fl = tid & 127;
    if (f >= p.F) return;
    const int rows = p.tn >> p.split_log, acc = DUAL ? 2 : 1, first = t0 + rank * rows, n = p.T - first < rows ? p.T - first : rows;
    constexpr int U = 4;
#pragma unroll 1
    for (int j0 = tid >> 7; j0 < n; j0 += 2 * U) {
        float v0[U], v1[U], r[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int j = j0 + 2 * k;
            v0[k] = v1[k] = 0.f;
            r[k] = j < n && p.residual ? from_bits16(p.residual[(long long)(first + j) * p.ld_res + f], HALF) : 0.f;
        }
#pragma unroll 1
        for (int i = 0; i < p.splits; ++i) {
            const float *src = red + (i * acc * rows + j0) * DT_FT + fl;
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (j0 + 2 * k < n) {
                    v0[k] += src[2 * k * DT_FT];
                    if (DUAL) v1[k] += src[(rows + 2 * k) * DT_FT];
                }
        }
#pragma unroll
        for (int k = 0; k < U; ++k)
            if (j0 + 2 * k < n) {
                const int t = first + j0 + 2 * k;
                const float y = dense_finish<DUAL, ACT>(p, v0[k], v1[k], b0, b1, f, t, col_blocks);
                out[(long long)t * p.ld_out + f] = to_bits16(y + r[k], HALF);
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
    const uint32_t a_bytes = ACC * DT_FT * 128, b_bytes = (uint32_t)p.tn * 128;
    const uint32_t stage_bytes = a_bytes + b_bytes;
    const uint32_t tile_bytes = (uint32_t)p.tn * ACC * DT_FT * 4;  // a whole partial tile, sent (over the stages) and received (behind them)
    float *red = reinterpret_cast<float *>(base + ((uint32_t)p.stages * stage_bytes > tile_bytes ? (uint32_t)p.stages * stage_bytes : tile_bytes));
    uint32_t cols = 32;
    while (cols < (uint32_t)p.tn * ACC) cols <<= 1;

    const int f = f0 + (int)(threadIdx.x & 127);  // this thread's output column: its lane of the accumulator
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
            tma_load_2d(a + 8192, ma, f0 + 64, r, &bar_full[slot]);
        } else {
            tma_load_2d(a, ma, r, f0, &bar_full[slot]);
            if (DUAL) tma_load_2d(a + 16384, &ma1, r, f0, &bar_full[slot]);
        }
        if (p.b_mn) {
            for (int i = 0; i < p.tn; i += 64) tma_load_2d(b + i * 128, mb, t0 + i, r, &bar_full[slot]);
        } else {
            tma_load_2d(b, mb, r, t0, &bar_full[slot]);
        }
    };
    const int ahead = k1 - k0 < p.stages ? k1 - k0 : p.stages;  // loads that need no free slot: under way before the rest is set up
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
            for (int i = 0; i < ahead; ++i) load(k0 + i, i);
        }
        __syncwarp();
    }
    if (p.splits > 1) cluster_arrive();  // (this CTA's barriers are ready)
    if (warp == 2) tmem_alloc(&tmem_base, cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base;

    if (warp == 0) {
        int slot = ahead == p.stages ? 0 : ahead;
        uint32_t phase = ahead == p.stages ? 1 : 0;
        for (int kb = k0 + ahead; kb < k1; ++kb) {
            if (!mbar_wait_abortable(&bar_free[slot], phase ^ 1, &abort_flag)) break;
            if (leader) load(kb, slot);
            __syncwarp();
            if (++slot == p.stages) slot = 0, phase ^= 1;
        }
    } else if (warp == 1) {
        // K-major: rows of 128 bytes, 8-row groups 1024 apart, 16 elements of the reduction 32 bytes on.
        // MN-major: 64-wide panels 8192 apart, 8 steps of the reduction 1024 apart, 16 of them 2048 on.
        const uint32_t a_step = (p.a_mn ? 2048 : 32) >> 4, b_step = (p.b_mn ? 2048 : 32) >> 4;
        const uint64_t ad0 = umma_desc_sw128(smem_u32(base), p.a_mn ? 8192 : 16, 1024);
        const uint64_t bd0 = umma_desc_sw128(smem_u32(base) + a_bytes, p.b_mn ? 8192 : 16, 1024);
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
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    umma_ss(tmem, ad + k * a_step, bd + k * b_step, p.idesc, kb > k0 || k > 0);
                    if (DUAL) umma_ss(tmem + p.tn, ad + (16384 >> 4) + k * a_step, bd + k * b_step, p.idesc, kb > k0 || k > 0);
                }
                umma_commit(&bar_free[slot]);
            }
            __syncwarp();
            if (++slot == p.stages) slot = 0, phase ^= 1;
        }
        if (ok && leader) umma_commit(&bar_done);
    }
    __syncwarp();
    const float b0 = p.bias0 && f < p.F ? load_bias(p.bias0, f, p.bias_fp32, HALF) : 0.f;  // (on its way while the products run)
    const float b1 = DUAL && p.bias1 && f < p.F ? load_bias(p.bias1, f, p.bias_fp32, HALF) : 0.f;
    bool ok = mbar_wait_abortable(&bar_done, 0, &abort_flag);
    tc_fence_after();
    if (p.splits > 1) {
        float *mine = reinterpret_cast<float *>(base);  // the stages have been read: this CTA's partial tile [accumulator][tn][128]
        if (ok) {
            const int q = warp & 3;
            for (int c = (warp >> 2) * 16; c < p.tn * ACC; c += 32) {
                const int tc = DUAL && c >= p.tn ? c - p.tn : c;
                if (t0 + tc >= p.T) continue;  // (warp-uniform)
                uint32_t v[16];
                tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + c, v);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) mine[(c + j) * DT_FT + q * 32 + lane] = __uint_as_float(v[j]);
            }
        }
        fence_proxy_async();
        tc_fence_before();
        __syncthreads();
        if (warp == 2) {
            tc_fence_after();
            tmem_relinquish();
            tmem_dealloc(tmem, cols);
        }
        __syncwarp();
        cluster_wait();  // every CTA of the cluster has its barriers: it can be sent to
        if (warp == 0 && lane < p.splits && ok) {
            const int left = p.T - t0 - lane * rows, n = left < 0 ? 0 : left < rows ? left : rows;  // rows that rank `lane` finishes
            const uint32_t bar = map_to_rank(smem_u32(&bar_red), lane);
#pragma unroll
            for (int a = 0; a < ACC; ++a)
                if (n > 0)
                    bulk_s2s(map_to_rank(smem_u32(red + (rank * ACC + a) * rows * DT_FT), lane), mine + (a * p.tn + lane * rows) * DT_FT,
                             (uint32_t)n * DT_FT * 4, bar);
        }
        __syncwarp();
        ok = mbar_wait_abortable(&bar_red, 0, &abort_flag) && ok;
        cluster_arrive();
    }
    if (ok) {
        switch (p.act) {
            case ACT_GELU: dense_epilogue<DUAL, ACT_GELU, HALF>(p, tmem, red, f, b0, b1, t0, group, rank); break;
            case ACT_SILU: dense_epilogue<DUAL, ACT_SILU, HALF>(p, tmem, red, f, b0, b1, t0, group, rank); break;
            case ACT_RELU: dense_epilogue<DUAL, ACT_RELU, HALF>(p, tmem, red, f, b0, b1, t0, group, rank); break;
            case ACT_SIGMOID: dense_epilogue<DUAL, ACT_SIGMOID, HALF>(p, tmem, red, f, b0, b1, t0, group, rank); break;
            default: dense_epilogue<DUAL, ACT_NONE, HALF>(p, tmem, red, f, b0, b1, t0, group, rank);
        }
    }
    __syncwarp();
    if (p.splits > 1) {
        cluster_wait();  // what this CTA sent has been received
    } else {
        tc_fence_before();
        __syncthreads();
        if (warp == 2) {
            tc_fence_after();
            tmem_relinquish();
            tmem_dealloc(tmem, cols);
        }
    }
}

}  // namespace pai
