// Host side of the feed-forward products: tensor maps, the choice of tile and split, the launches.
#pragma once
#include "dense_pair.cuh"
#include "dense_tile.cuh"
#include "dense_vec.cuh"

namespace pai {

inline long long dense_ld16(long long cols) { return (cols + 7) / 8 * 8; }  // row pitch of a 16-bit workspace matrix

// Map of a [rows, inner] matrix of 16-bit elements with row pitch `ld` elements, boxes of box_rows rows x 64 columns (128-byte swizzle) or 32 (64-byte
// swizzle); outside reads as 0.
static int make_map_16(CUtensorMap *map, const void *base, long long inner, long long rows, long long ld, int box_rows, int half, int box_cols = 64) {
    EncodeTiledFn enc = get_encode_tiled();
    if (!enc) return (int)PAI_ERR_UNSUPPORTED;
    cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)(rows > 1 ? ld : dense_ld16(inner)) * 2};
    cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = enc(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(base), dims, strides, box,
                     estr, CU_TENSOR_MAP_INTERLEAVE_NONE, box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : (int)PAI_ERR_UNSUPPORTED;
}

// Launch as a programmatic dependent of what is on the stream (common.cuh), in clusters of `cluster` CTAs if it is more than 1; cluster 0: in
// order.  A kernel that lives on plain loads goes in order behind the products: brought onto their SMs early it also inherits their split of
// the SM's memory, which leaves it next to no L1 for loads in flight (joining 32 tiles of 512 x 256: 33 us for 8; a gated training step of
// 16384 x 512 x 2048: 245 us for 230).
template <typename... P, typename... A>
static int dense_launch_kernel(void (*kernel)(P...), dim3 grid, int block, int smem, cudaStream_t st, int cluster, const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : cluster;
    return (int)cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

struct DenseOperand {       // a matrix of 16-bit elements
    const void *p;
    long long ld;
};

// One product: out[t, f] (+ epilogue); `a[i]`, `b[i]` the operand pairs, `dual` / `segs` / `groups` as in dense_tile.cuh.
struct DenseProduct {
    DenseOperand a[2], b[2];
    int a_mn, b_mn, dual, segs, groups;
    long long F, T, R;
    void *out[2];
    long long ld_out;
    const void *bias[2];
    int bias_fp32;
    const void *residual;
    long long ld_res;
    void *save[2];
    int act, half;
    DenseColsum colsum;        // bias gradients that the product's kernel finishes
    float *part;               // workspace of a split reduction in the pair kernel (dense_pair_choose), or NULL: no split
};

// Test-only overrides of the choices below (0: none): kernel 1 = tile, 2 = pair (3 = vec, which takes no shape); tile height / accumulator columns; split.
struct DenseTune {
    int kernel, width, splits;
};
static DenseTune g_dense_tune;

// The kernel and its shape are the ones with the lowest estimated time, in microseconds: models with coefficients fitted to 699 measurements of all
// shapes at 19 sizes from 16 x 512 x 2048 to 16384 x 512 x 2048, one product after another on a stream (r.m.s. 9 and 7 %; the cost per split
// came later, from reductions of up to 65536).  The choice is within 10 % of the best shape measured on all of 83 products.
struct DenseChoice {
    int pair, width, splits;   // width: rows t of a tile (tile kernel), accumulator columns (pair kernel)
    double cost;
};

// Tile kernel: start and end; per reduction block the instructions of its loads and MMAs; per row of the tile the epilogue, shared by
// the CTAs of a split reduction but with its exchange.  Clusters of 4 and 8 leave SMs of a GPC unused.
static DenseChoice dense_tile_choose(const DenseProduct &d, int sms) {
    const long long kb = (d.R + DT_BK - 1) / DT_BK * d.segs;
    const int acc = d.dual ? 2 : 1, least = d.b_mn ? 64 : 16;
    DenseChoice best = {0, 64, 1, 1e300};
    for (int tn = least; tn <= (d.dual ? 128 : 256); tn *= 2) {
        if (tn > least && tn / 2 >= d.T && g_dense_tune.width == 0) break;
        if (g_dense_tune.kernel == 1 && g_dense_tune.width && tn != g_dense_tune.width) continue;
        const long long tiles = (d.F + DT_FT - 1) / DT_FT * ((d.T + tn - 1) / tn) * d.groups;
        for (int splits = 1; splits <= 8 && splits <= kb; splits *= 2) {
            if (g_dense_tune.kernel == 1 && g_dense_tune.splits && splits != g_dense_tune.splits) continue;
            if (splits > 1 && tn * acc > 128) continue;  // (the partial rows' buffer)
            const long long room = splits == 8 ? sms * 3 / 4 : splits == 4 ? sms * 8 / 9 : sms;
            const double rounds = (double)((tiles * splits + room - 1) / room), blocks = (double)((kb + splits - 1) / splits), w = tn * acc;
            const double cta = 0.81 + blocks * (0.426 + 0.00083 * w + (d.dual ? 0.156 : 0.0)) + 0.0243 * w / splits + (splits > 1 ? 0.49 + 0.036 * w : 0.0);
            const double t = 1.8 + (rounds > 1 ? 1.08 * rounds : 1.0) * cta;
            if (t < best.cost) best = {0, tn, splits, t};
        }
    }
    return best;
}

// Pair kernel: start and end; per tile the products of its reduction and what of the epilogue they do not cover; a split reduction writes and
// reads fp32 tiles and adds a launch.
static DenseChoice dense_pair_choose(const DenseProduct &d, int sms, bool may_split) {
    const long long kb = (d.R + DP_BK - 1) / DP_BK * d.segs;
    const double out = 1e-6 * (double)d.F * (double)d.T * d.groups;
    DenseChoice best = {1, 256, 1, 1e300};
    for (int bn = d.dual ? 256 : 128; bn <= 256; bn *= 2) {
        if (g_dense_tune.kernel == 2 && g_dense_tune.width && bn != g_dense_tune.width) continue;
        const int fw = d.dual ? bn / 2 : bn;
        const long long tiles = (d.F + fw - 1) / fw * ((d.T + 255) / 256) * d.groups;
        for (int splits = 1; splits <= (may_split ? 64 : 1) && splits * 4 <= (kb > 4 ? kb : 4); ++splits) {
            if (g_dense_tune.kernel == 2 && g_dense_tune.splits && may_split && splits != g_dense_tune.splits) continue;
            if (splits > 1 && tiles * splits > sms / 2 && g_dense_tune.splits == 0) break;  // (a second round of short items costs more than it saves)
            const double rounds = (double)((tiles * splits + sms / 2 - 1) / (sms / 2)), blocks = (double)((kb + splits - 1) / splits);
            const double tile = bn == 256 ? 0.29 * blocks + 0.46 : 0.237 * blocks;
            const double t = 3.85 + rounds * tile + 0.287 * out + (splits > 1 ? 1.65 + splits * (0.16 + 1.54 * out) : 0.0);
            if (t < best.cost) best = {1, bn, splits, t};
        }
    }
    return best;
}

static DenseChoice dense_choose(const DenseProduct &d, int sms, bool may_split) {
    const DenseChoice a = dense_tile_choose(d, sms), b = dense_pair_choose(d, sms, may_split);
    if (g_dense_tune.kernel) return g_dense_tune.kernel == 2 ? b : a;  // (3: what the vec kernel does not run)
    return b.cost < a.cost ? b : a;
}

template <bool DUAL, int HALF>
static int dense_tile_launch_as(const CUtensorMap (&m)[4], const DenseTileParams &p, dim3 grid, int smem, cudaStream_t st) {
    static bool attr_done[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        cudaError_t e = cudaFuncSetAttribute(dense_tile_kernel<DUAL, HALF>, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024);
        if (e != cudaSuccess) return (int)e;
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    return dense_launch_kernel(dense_tile_kernel<DUAL, HALF>, grid, DT_THREADS, smem, st, p.splits, m[0], m[1], m[2], m[3], p);
}

static uint32_t dense_idesc(int m, int n, const DenseProduct &d, int m_mn, int n_mn) {
    return (umma_idesc_bf16(m, n, m_mn != 0, n_mn != 0) & ~((7u << 7) | (7u << 10))) | (d.half ? 0u : (1u << 7) | (1u << 10));
}

static int dense_tile_launch(const DenseProduct &d, const DenseChoice &c, int sms, cudaStream_t st) {
    const int tn = c.width, splits = c.splits;
    DenseTileParams p = {};
    p.out0 = d.out[0], p.out1 = d.out[1];
    p.bias0 = d.bias[0], p.bias1 = d.bias[1];
    p.residual = (const unsigned short *)d.residual;
    p.save0 = (float *)d.save[0], p.save1 = (float *)d.save[1];
    p.ld_out = d.ld_out, p.ld_res = d.ld_res;
    p.F = (int)d.F, p.T = (int)d.T;
    const long long f_tiles = (d.F + DT_FT - 1) / DT_FT, t_tiles = (d.T + tn - 1) / tn;  // (f_tiles <= 2^13: widths are limited)
    p.splits = splits, p.split_log = splits == 8 ? 3 : splits == 4 ? 2 : splits == 2 ? 1 : 0, p.tn = tn;
    p.kb_seg = (int)((d.R + DT_BK - 1) / DT_BK), p.kb_total = p.kb_seg * d.segs;
    p.tail = d.R % DT_BK > 0 && d.R % DT_BK <= 64;
    p.colsum = d.colsum;
    p.a_mn = d.a_mn, p.b_mn = d.b_mn;
    p.act = d.act, p.bias_fp32 = d.bias_fp32;
    p.idesc = dense_idesc(128, tn, d, d.a_mn, d.b_mn);
    const long long ctas = f_tiles * t_tiles * d.groups * splits;
    if (t_tiles * splits > 0x7fffffffll) return (int)PAI_ERR_BAD_SHAPE;
    const int stage = (d.dual ? 2 : 1) * DT_FT * 256 + tn * 256, kb_cta = (p.kb_total + splits - 1) / splits;
    const int tile = tn * DT_FT * 4 * (d.dual ? 2 : 1), red = splits > 1 ? tile : 0;  // an fp32 tile; partial rows sent here
    int stages = ((ctas > sms && 2 * stage + red <= 108 * 1024 ? 108 : 216) * 1024 - red) / stage;  // two CTAs per SM if two stages each fit
    stages = stages > DT_MAX_STAGES ? DT_MAX_STAGES : stages;
    stages = stages > kb_cta ? kb_cta : stages;
    p.stages = stages = stages < 1 ? 1 : stages;
    // (the stages also hold the CTA's own partial tile)
    const int smem = (stages * stage > tile ? stages * stage : tile) + red + 1024;
    const dim3 grid((unsigned)(t_tiles * splits), (unsigned)f_tiles, d.groups);
    CUtensorMap m[4];
    for (int i = 0; i < 2; ++i) {
        const DenseOperand &a = d.a[i].p ? d.a[i] : d.a[0], &b = d.b[i].p ? d.b[i] : d.b[0];
        if (i == 1 && !d.a[1].p) m[1] = m[0];
        else if (int e = d.a_mn ? make_map_16(&m[i], a.p, d.F, d.R, a.ld, DT_BK, d.half) : make_map_16(&m[i], a.p, d.R, d.F, a.ld, DT_FT, d.half)) return e;
        if (i == 1 && !d.b[1].p) m[3] = m[2];
        else if (int e = d.b_mn ? make_map_16(&m[2 + i], b.p, d.T, d.R, b.ld, DT_BK, d.half) : make_map_16(&m[2 + i], b.p, d.R, d.T, b.ld, tn, d.half)) return e;
    }
    if (d.half) return d.dual ? dense_tile_launch_as<true, 1>(m, p, grid, smem, st) : dense_tile_launch_as<false, 1>(m, p, grid, smem, st);
    return d.dual ? dense_tile_launch_as<true, 0>(m, p, grid, smem, st) : dense_tile_launch_as<false, 0>(m, p, grid, smem, st);
}

// map of an operand as MMA rows (`rows` of them, `box` per load): reduction-contiguous or not
static int make_operand_map(CUtensorMap *m, const DenseOperand &o, int mn, long long rows, long long R, int box, int half) {
    return mn ? make_map_16(m, o.p, rows, R, o.ld, 64, half) : make_map_16(m, o.p, R, rows, o.ld, box, half);
}

template <int MODE, int HALF, int FLAGS>
static int dense_pair_launch_as(const CUtensorMap (&m)[6], const DensePairParams &p, int ctas, cudaStream_t st) {
    static bool attr_done[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        cudaError_t e = cudaFuncSetAttribute(dense_pair_kernel<MODE, HALF, FLAGS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(DensePairSmem));
        if (e != cudaSuccess) return (int)e;
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    return dense_launch_kernel(dense_pair_kernel<MODE, HALF, FLAGS>, dim3(ctas), DP_THREADS, (int)sizeof(DensePairSmem), st, 1, m[0], m[1], m[2], m[3],
                               m[4], m[5], p);
}

template <int HALF>
static int dense_pair_launch_half(const CUtensorMap (&m)[6], const DensePairParams &p, int dual, int flags, int ctas, cudaStream_t st) {
    if (dual) {
        if (flags == DP_ANY) return dense_pair_launch_as<DP_GATED, HALF, DP_ANY>(m, p, ctas, st);
        return flags ? dense_pair_launch_as<DP_GATED, HALF, DP_SAVE>(m, p, ctas, st) : dense_pair_launch_as<DP_GATED, HALF, 0>(m, p, ctas, st);
    }
    switch (flags) {
        case 0: return dense_pair_launch_as<DP_LINEAR, HALF, 0>(m, p, ctas, st);
        case DP_RESIDUAL: return dense_pair_launch_as<DP_LINEAR, HALF, DP_RESIDUAL>(m, p, ctas, st);
        case DP_SAVE: return dense_pair_launch_as<DP_LINEAR, HALF, DP_SAVE>(m, p, ctas, st);
        case DP_RESIDUAL | DP_SAVE: return dense_pair_launch_as<DP_LINEAR, HALF, DP_RESIDUAL | DP_SAVE>(m, p, ctas, st);
        default: return dense_pair_launch_as<DP_LINEAR, HALF, DP_ANY>(m, p, ctas, st);
    }
}

// (in the roles of DenseProduct the pair kernel's rows are t, its columns f: its A is `b`, its B is `a`)
static int dense_pair_launch(const DenseProduct &d, const DenseChoice &c, int sms, cudaStream_t st) {
    if (d.groups > 1 && c.splits == 1) {  // two whole products: one output map each
        for (int g = 0; g < d.groups; ++g) {
            DenseProduct e = d;
            e.groups = 1;
            e.b[0] = d.b[g], e.b[1] = {nullptr, 0};
            e.out[0] = d.out[g], e.out[1] = nullptr;
            if (g > 0) e.colsum = {};
            if (int r = dense_pair_launch(e, c, sms, st)) return r;
        }
        return 0;
    }
    DensePairParams p = {};
    const int fw = d.dual ? c.width / 2 : c.width;
    p.out0 = (unsigned short *)d.out[0];
    p.residual = (const unsigned short *)d.residual;
    p.bias0 = d.bias[0], p.bias1 = d.bias[1], p.bias_fp32 = d.bias_fp32;
    p.save0 = (uint8_t *)d.save[0], p.save1 = (uint8_t *)d.save[1];
    p.save_f32 = d.half;
    p.save_exps = (long long)saved_blocks(d.T, (int)d.F) * 2048;
    p.part = d.part;
    p.colsum = d.colsum;
    p.ld_out = d.ld_out, p.ld_res = d.ld_res;
    p.T = (int)d.T, p.F = (int)d.F, p.bn = c.width;
    p.t_tiles = (int)((d.T + 255) / 256), p.f_tiles = (int)((d.F + fw - 1) / fw), p.groups = d.groups, p.splits = c.splits;
    p.kb_seg = (int)((d.R + DP_BK - 1) / DP_BK), p.kb_total = p.kb_seg * d.segs;
    p.a_mn = d.b_mn, p.b_mn = d.a_mn, p.act = d.act;
    p.idesc = dense_idesc(256, c.width, d, d.b_mn, d.a_mn);
    const long long items = (long long)p.t_tiles * p.f_tiles * p.groups * p.splits;
    if (items > 0x3fffffffll) return (int)PAI_ERR_BAD_SHAPE;
    CUtensorMap m[6];
    for (int i = 0; i < 2; ++i) {
        if (i == 1 && !d.b[1].p) m[1] = m[0];
        else if (int e = make_operand_map(&m[i], d.b[i], d.b_mn, d.T, d.R, 128, d.half)) return e;
        if (i == 1 && !d.a[1].p) m[3] = m[2];
        else if (int e = make_operand_map(&m[2 + i], d.a[i], d.a_mn, d.F, d.R, c.width / 2, d.half)) return e;
    }
    m[4] = m[5] = m[0];
    const bool partial = c.splits > 1;
    p.tma_out = !partial && ((uintptr_t)d.out[0] & 15) == 0 && (d.T == 1 || (d.ld_out & 7) == 0);
    if (p.tma_out)
        if (int e = make_map_16(&m[4], d.out[0], d.F, d.T, d.ld_out, 32, d.half, 32)) return e;
    p.tma_res = d.residual && ((uintptr_t)d.residual & 15) == 0 && (d.T == 1 || ((d.ld_res & 7) == 0 && d.ld_res >= d.F));
    if (p.tma_res)
        if (int e = make_map_16(&m[5], d.residual, d.F, d.T, d.ld_res, 32, d.half, 32)) return e;
    const int ctas = 2 * (int)(items < sms / 2 ? items : sms / 2);
    if (partial) {
        if (int e = d.half ? dense_pair_launch_as<DP_PARTIAL, 1, 0>(m, p, ctas, st) : dense_pair_launch_as<DP_PARTIAL, 0, 0>(m, p, ctas, st)) return e;
        const size_t blocks = saved_blocks(d.T, (int)d.F);
        return dense_launch_kernel(dense_reduce_kernel, dim3((unsigned)blocks, d.groups), 256, 0, st, 0, d.part, d.out[0], d.out[1], p.T, p.F, d.ld_out,
                                   d.groups, c.splits, d.half);
    }
    const int any = !p.tma_out || (d.residual && !p.tma_res) ? DP_ANY : 0;
    const int flags = any ? any : (d.residual ? DP_RESIDUAL : 0) | (d.save[0] ? DP_SAVE : 0);
    return d.half ? dense_pair_launch_half<1>(m, p, d.dual, flags, ctas, st) : dense_pair_launch_half<0>(m, p, d.dual, flags, ctas, st);
}

static int dense_launch(const DenseProduct &d, int sms, cudaStream_t st) {
    const DenseChoice c = dense_choose(d, sms, d.part != nullptr);
    return c.pair ? dense_pair_launch(d, c, sms, st) : dense_tile_launch(d, c, sms, st);
}

// ---- up to eight tokens ---------------------------------------------------------------------------------------------
template <bool DUAL, int ACT, int TT>
static int dense_vec_as(const DenseVecParams &p, int half, unsigned grid, cudaStream_t st) {
    return half ? dense_launch_kernel(dense_vec_kernel<DUAL, ACT, TT, 1>, dim3(grid), DV_WARPS * 32, 0, st, 1, p)
                : dense_launch_kernel(dense_vec_kernel<DUAL, ACT, TT, 0>, dim3(grid), DV_WARPS * 32, 0, st, 1, p);
}
template <bool DUAL, int ACT>
static int dense_vec_tokens(const DenseVecParams &p, int half, unsigned grid, cudaStream_t st) {
    if (p.T <= 1) return dense_vec_as<DUAL, ACT, 1>(p, half, grid, st);
    if (p.T <= 2) return dense_vec_as<DUAL, ACT, 2>(p, half, grid, st);
    if (p.T <= 4) return dense_vec_as<DUAL, ACT, 4>(p, half, grid, st);
    return dense_vec_as<DUAL, ACT, 8>(p, half, grid, st);
}
template <bool DUAL>
static int dense_vec_act(const DenseVecParams &p, int act, int half, cudaStream_t st) {
    const int per_cta = DV_WARPS * (DUAL ? 1 : 2);
    const unsigned grid = (unsigned)((p.N + per_cta - 1) / per_cta);
    switch (act) {
        case ACT_GELU: return dense_vec_tokens<DUAL, ACT_GELU>(p, half, grid, st);
        case ACT_SILU: return dense_vec_tokens<DUAL, ACT_SILU>(p, half, grid, st);
        case ACT_RELU: return dense_vec_tokens<DUAL, ACT_RELU>(p, half, grid, st);
        case ACT_SIGMOID: return dense_vec_tokens<DUAL, ACT_SIGMOID>(p, half, grid, st);
        default: return dense_vec_tokens<DUAL, ACT_NONE>(p, half, grid, st);
    }
}
static bool dense_uses_vec(long long T) { return T <= DV_MAX_TOKENS && (g_dense_tune.kernel == 0 || g_dense_tune.kernel == 3); }
static int dense_vec_launch(const DenseProduct &d, cudaStream_t st) {
    DenseVecParams p = {};
    p.x = (const unsigned short *)d.b[0].p, p.w0 = (const unsigned short *)d.a[0].p, p.w1 = (const unsigned short *)d.a[1].p;
    p.ld_x = d.b[0].ld, p.ld_w0 = d.a[0].ld, p.ld_w1 = d.a[1].ld;
    p.bias0 = d.bias[0], p.bias1 = d.bias[1], p.bias_fp32 = d.bias_fp32;
    p.residual = (const unsigned short *)d.residual, p.ld_res = d.ld_res;
    p.out = (unsigned short *)d.out[0], p.ld_out = d.ld_out;
    p.save0 = (float *)d.save[0], p.save1 = (float *)d.save[1];
    p.T = (int)d.T, p.N = (int)d.F, p.K = (int)d.R;
    return d.dual ? dense_vec_act<true>(p, d.act, d.half, st) : dense_vec_act<false>(p, d.act, d.half, st);
}

// The products as problems (sizes only): what the saved buffer and the workspace are sized for, and what runs.
static DenseProduct dense_forward_product(long long M, int N, int K, int gated) {
    DenseProduct d = {};
    d.dual = gated, d.segs = 1, d.groups = 1;
    d.F = N, d.T = M, d.R = K;
    return d;
}
static DenseProduct dense_weight_product(long long M, int N, int K, int groups) {
    DenseProduct d = {};
    d.a_mn = 1, d.b_mn = 1, d.segs = 1, d.groups = groups;
    d.F = K, d.T = N, d.R = M;
    return d;
}
// the form of the saved pre-activations: fp16 with exponents where the pair kernel runs on bf16, fp32 otherwise
static bool dense_saves_f32(long long M, int N, int K, int gated, int half, int sms) {
    return half || dense_uses_vec(M) || !dense_choose(dense_forward_product(M, N, K, gated), sms, false).pair;
}
static size_t dense_saved_matrix(long long M, int N, int K, int gated, int half, int sms) {
    return dense_saves_f32(M, N, K, gated, half, sms) ? saved_bytes_f32(M, N) : saved_bytes_f16(M, N);
}

// ---- the two operators ----------------------------------------------------------------------------------------------
static int dense_forward(const DenseOperand &x, const DenseOperand (&w)[2], const void *const (&bias)[2], int bias_fp32, const DenseOperand &residual,
                         void *y, long long ldy, void *saved, long long M, int N, int K, int act, int half, int sms, cudaStream_t st) {
    const bool gated = w[1].p != nullptr;
    DenseProduct d = dense_forward_product(M, N, K, gated);
    d.a[0] = w[0], d.a[1] = w[1];
    d.b[0] = x;
    d.out[0] = y, d.ld_out = ldy;
    d.bias[0] = bias[0], d.bias[1] = bias[1], d.bias_fp32 = bias_fp32;
    d.residual = residual.p, d.ld_res = residual.ld;
    d.save[0] = saved;
    d.save[1] = saved && gated ? (char *)saved + dense_saved_matrix(M, N, K, gated, half, sms) : nullptr;
    d.act = act, d.half = half;
    return dense_uses_vec(M) ? dense_vec_launch(d, st) : dense_launch(d, sms, st);
}

// Strips of the elementwise pass: about four CTAs of 256 threads per SM, at least 64 rows each.
inline int dense_strip_rows(long long M, int N) {
    const long long col_ctas = (N + 255) / 256, want = 592 / col_ctas > 0 ? 592 / col_ctas : 1;
    long long strip = (M + want - 1) / want;
    strip = strip < 64 ? 64 : (strip + 7) / 8 * 8;
    return (int)strip;
}
inline long long dense_strips(long long M, int N) {
    const int s = dense_strip_rows(M, N);
    return (M + s - 1) / s;
}
inline size_t align256(size_t b) { return (b + 255) / 256 * 256; }
// workspace: the 16-bit gradient(s) of the pre-activations, the strips' column sums, the fp32 tiles of a split weight gradient
inline size_t dense_d_bytes(long long M, int N) { return align256((size_t)M * dense_ld16(N) * 2); }
inline size_t dense_part_bytes(long long M, int N) { return align256((size_t)dense_strips(M, N) * N * 4); }
static size_t dense_split_bytes(long long M, int N, int K, int mats, int sms) {
    size_t most = 0;
    for (int g = 1; g <= mats; ++g) {  // (one of the two weight gradients alone may split further)
        const DenseChoice c = dense_choose(dense_weight_product(M, N, K, g), sms, true);
        const size_t b = c.pair && c.splits > 1 ? (size_t)c.splits * g * saved_bytes_f32(N, K) : 0;
        most = b > most ? b : most;
    }
    return most;
}
static size_t dense_bwd_workspace(long long M, int N, int K, int mats, int sms) {
    return mats * (dense_d_bytes(M, N) + dense_part_bytes(M, N)) + dense_split_bytes(M, N, K, mats, sms);
}

template <bool DUAL, int ACT>
static int dense_bwd_elem_as(const DenseBwdElemParams &p, int half, bool f32, dim3 grid, cudaStream_t st) {
    if (half) return dense_launch_kernel(dense_bwd_elem_kernel<DUAL, ACT, 1, true>, grid, 256, 0, st, 0, p);
    return f32 ? dense_launch_kernel(dense_bwd_elem_kernel<DUAL, ACT, 0, true>, grid, 256, 0, st, 0, p)
               : dense_launch_kernel(dense_bwd_elem_kernel<DUAL, ACT, 0, false>, grid, 256, 0, st, 0, p);
}
template <bool DUAL>
static int dense_bwd_elem_act(const DenseBwdElemParams &p, int act, int half, bool f32, dim3 grid, cudaStream_t st) {
    switch (act) {
        case ACT_GELU: return dense_bwd_elem_as<DUAL, ACT_GELU>(p, half, f32, grid, st);
        case ACT_SILU: return dense_bwd_elem_as<DUAL, ACT_SILU>(p, half, f32, grid, st);
        case ACT_RELU: return dense_bwd_elem_as<DUAL, ACT_RELU>(p, half, f32, grid, st);
        case ACT_SIGMOID: return dense_bwd_elem_as<DUAL, ACT_SIGMOID>(p, half, f32, grid, st);
        default: return dense_bwd_elem_as<DUAL, ACT_NONE>(p, half, f32, grid, st);
    }
}
static int dense_bwd_elem_launch(const DenseBwdElemParams &p, bool gated, int act, int half, bool f32, unsigned strips, cudaStream_t st) {
    const dim3 grid((p.N + 255) / 256, strips);
    return gated ? dense_bwd_elem_act<true>(p, act, half, f32, grid, st) : dense_bwd_elem_act<false>(p, act, half, f32, grid, st);
}

static int dense_backward(const DenseOperand &dy, const DenseOperand &x, const DenseOperand (&w)[2], const void *saved, void *dx, long long lddx,
                          void *const (&dw)[2], void *const (&db)[2], int bias_fp32, void *workspace, long long M, int N, int K, int act, int half,
                          int sms, cudaStream_t st) {
    const bool gated = w[1].p != nullptr;
    const int mats = gated ? 2 : 1;
    const bool elementwise = gated || act != ACT_NONE;
    const bool products = dx || dw[0] || dw[1];
    DenseOperand dz[2] = {dy, {nullptr, 0}};
    char *ws = (char *)workspace;
    const long long strips = dense_strips(M, N);
    DenseBwdElemParams p = {};
    p.dy = (const unsigned short *)dy.p, p.ld_dy = dy.ld;
    p.vec_dy = ((uintptr_t)dy.p & 15) == 0 && (dy.ld & 7) == 0;
    p.M = M, p.N = N, p.strip = dense_strip_rows(M, N);
    const bool f32 = dense_saves_f32(M, N, K, gated, half, sms);
    if (elementwise) {
        p.save0 = (const uint8_t *)saved;
        p.save1 = gated ? (const uint8_t *)saved + dense_saved_matrix(M, N, K, gated, half, sms) : nullptr;
        p.save_exps = saved_blocks(M, N) * 2048;
        if (products) {
            p.ld_d = dense_ld16(N);
            p.d0 = (unsigned short *)ws;
            p.d1 = gated ? (unsigned short *)(ws + dense_d_bytes(M, N)) : nullptr;
            dz[0] = {p.d0, p.ld_d}, dz[1] = {p.d1, p.ld_d};
        }
    }
    if (db[0] || db[1]) {
        p.part0 = (float *)(ws + mats * dense_d_bytes(M, N));
        p.part1 = gated ? p.part0 + dense_part_bytes(M, N) / 4 : nullptr;
    }
    if ((elementwise && products) || p.part0) {
        if (int e = dense_bwd_elem_launch(p, gated, act, half, f32, (unsigned)strips, st)) return e;
    }
    DenseColsum colsum = {};
    if (p.part0) {
        colsum = {{db[0] ? p.part0 : nullptr, db[1] ? p.part1 : nullptr}, {db[0], db[1]}, N, (int)strips, bias_fp32};
        if (!products) {
            const dim3 grid((N + 31) / 32);
            return half ? dense_launch_kernel(dense_colsum_kernel<1>, grid, 32, 0, st, 1, colsum)
                        : dense_launch_kernel(dense_colsum_kernel<0>, grid, 32, 0, st, 1, colsum);
        }
    }
    if (dx) {
        DenseProduct d = {};
        d.a[0] = w[0], d.a[1] = w[1], d.a_mn = 1;
        d.b[0] = dz[0], d.b[1] = dz[1];
        d.segs = mats, d.groups = 1;
        d.F = K, d.T = M, d.R = N;
        d.out[0] = dx, d.ld_out = lddx, d.half = half;
        d.colsum = colsum;
        colsum = {};
        if (int e = dense_launch(d, sms, st)) return e;
    }
    if (dw[0] || dw[1]) {
        DenseProduct d = dense_weight_product(M, N, K, dw[0] && dw[1] ? 2 : 1);
        d.a[0] = x;
        d.b[0] = dw[0] ? dz[0] : dz[1], d.out[0] = dw[0] ? dw[0] : dw[1];
        if (d.groups == 2) d.b[1] = dz[1], d.out[1] = dw[1];
        d.ld_out = K, d.half = half;
        d.colsum = colsum;
        d.part = (float *)(ws + mats * (dense_d_bytes(M, N) + dense_part_bytes(M, N)));
        if (int e = dense_launch(d, sms, st)) return e;
    }
    return 0;
}

static int dense_copy_rows(const DenseCopyParams &p, int count, int sms, cudaStream_t st) {
    long long most = 0;
    for (int i = 0; i < count; ++i) most = p.rows[i] * ((p.cols[i] + 7) / 8) > most ? p.rows[i] * ((p.cols[i] + 7) / 8) : most;
    if (most == 0) return 0;
    long long blocks = (most + 255) / 256;
    if (blocks > (long long)sms * 16) blocks = (long long)sms * 16;
    return dense_launch_kernel(dense_copy_rows_kernel, dim3((unsigned)blocks, count), 256, 0, st, 1, p);
}

}  // namespace pai
