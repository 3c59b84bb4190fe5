// Product of two matrices of block-scaled 4-bit numbers (quant4.cuh) on sm_100a: C = epilogue(alpha * A[M,K] * W[N,K]^T). The tensor cores take the
// codes and the scales as they lie in memory: tcgen05.mma kind::mxf4 (MX4, a scale per 32) and kind::mxf4nvf4 (NV4, a scale per 16) multiply
// the 64 products of a k step by their blocks' scales and sum in fp32 in TMEM. Every product and its scaling is exact; only the sums round.
//
// The schedule is that of the fp16 product next door (gemm_sm100.cuh): persistent CTAs, one warp loads by TMA, one issues, sixteen run the epilogue of one
// tile under the main loop of the next. What differs: a k step in shared memory holds 256 columns (128 bytes) of each operand, plus their scales
// (2 KB per 128 rows for NV4, 1 KB for MX4), which tcgen05.cp copies to TMEM in front of the step's products, four lanes' quarters at a time.
//
// Two shapes. Single: one CTA per 128 x 128 tile. PAIR: two CTAs on a 256 x 256 tile (cta_group::2): each loads its 128 rows of A, half of the W rows, the
// scales of its rows and of ALL columns of the tile, and keeps its half of the accumulator. Two accumulators of 256 columns fill TMEM and leave no
// room for scales, so they overlap: the first lies in columns [0, 256), the second in [128, 384), the scales behind them. The epilogue drains the 128
// columns that both own first, and then the next tile's products begin; until then the tensor pipe waits, some 1000 clocks per tile. (Pairs on 192 columns, which
// have two whole accumulators beside the scales, wait for their loads instead: with eight epilogue warps N 8192, K 2048, M 4096
// took 37.3 us against 36.0, K 8192, N 2048 32.6 against 28.6.)
//
// What bounds it: a step of a pair takes the products' 512 clocks (490-510 from one to the next by the clock counter), so a long k range runs at the pipe's rate
// for the clock that the power cap leaves: 8192^3 back to back 229 us at 1.36 GHz and 990 W (4.8 PFLOP/s; 199 us, 5.5, before the clock falls), M 4096, N 2048,
// K 8192 28.6 us. Short ranges add the waits between tiles: M 4096, N 8192, K 2048 32.4 us, of which the products take 24 at 1.65 GHz.
#pragma once
#include "gemm_sm100.cuh"   // gelu, elect_one, pack16
#include "quant4.cuh"

namespace kb {

constexpr int EPI_GELU4 = 5;                               // C leaves in 4 bits: codes and scales of gelu(alpha * acc)

constexpr int G4_K = 256;                                  // columns of a k step: 128 bytes of codes
constexpr int G4_STAGES = 5;
constexpr int G4_SF_OFF = 32768;                           // scales of a stage: A's 128 rows, then W's
constexpr int G4_STAGE_BYTES = G4_SF_OFF + 6144;
// Sixteen epilogue warps, four per TMEM lane quarter, with 32 columns at a time: GELU and quantisation are ~17 instructions per element, and eight warps kept the
// issue slots 42 % busy (M 4096, N 8192, K 2048 into GELU in 4 bits: 8 warps 44.0 us, 16, with both chunks' loads in front, 41.7).
constexpr int G4_EPI_WARPS = 16, G4_THREADS = 32 * (G4_EPI_WARPS + 4);   // last warpgroup: MMA issue, TMA loads, two idle
constexpr int G4_STAGING_WARP = 2048;                      // a box of 32 rows x 64 bytes on its way out
constexpr int G4_SMEM = G4_STAGES * G4_STAGE_BYTES + G4_EPI_WARPS * G4_STAGING_WARP + 1024 + 1024;
static_assert(G4_SMEM <= 232448, "shared memory of a thread block");

struct Gemm4Params {
    int M, N, K;                   // K: columns of the k steps that exist in memory (a multiple of 32)
    int tiles_m, tiles_n;
    float alpha;
    void* C;
    int ldc;
    const float* gate;             // EPI_RESID: C[r, c] += gate[c] * alpha * acc (null = 1)
    uint8_t* codes;                // EPI_GELU4
    uint8_t* scales;
    int ld_codes, pieces;
    uint32_t* status;
};

struct alignas(64) Gemm4Maps {
    CUtensorMap a, w;              // codes: box 128 bytes x 128 rows
    CUtensorMap sa, sw;            // scales: [row block][piece][512 bytes], box of one step's pieces of one row block
    CUtensorMap c;                 // output
};

enum { G4BAR_FULL = 0, G4BAR_EMPTY = G4_STAGES, G4BAR_ACC_FULL = 2 * G4_STAGES, G4BAR_ACC_EMPTY = 2 * G4_STAGES + 2, G4BAR_COUNT = 2 * G4_STAGES + 4 };

// Instruction descriptor of the block-scaled kinds: W's scale byte in bits [4, 6), A and B formats at 7 and 10 (1 = e2m1), N >> 3 in
// [17, 23), scales' type in bit 23 (0 = E4M3, 1 = E8M0), M >> 4 in [24, 29), A's scale byte in [29, 31). Both operands K-major.
__host__ __device__ constexpr uint32_t idesc_f4(bool e8m0, int M, int N, int sf_byte) {
    return ((uint32_t)sf_byte << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)e8m0 << 23) | ((uint32_t)(M >> 4) << 24) |
           ((uint32_t)sf_byte << 29);
}
// D[tmem] (+)= scaled A[smem] * scaled B[smem], 64 columns; scales at sa, sb in TMEM
template <int FMT, bool PAIR>
__device__ __forceinline__ void mma_f4(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
#define KB_MMA4(group, kind)                                                                                                         \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                                                   \
                 "tcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d_tmem), "l"(adesc),   \
                 "l"(bdesc), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)                                                           \
                 : "memory")
    if constexpr (FMT == FMT_MX4) {
        if constexpr (PAIR) KB_MMA4("2", "mxf4.block_scale.scale_vec::2X"); else KB_MMA4("1", "mxf4.block_scale.scale_vec::2X");
    } else {
        if constexpr (PAIR) KB_MMA4("2", "mxf4nvf4.block_scale.scale_vec::4X"); else KB_MMA4("1", "mxf4nvf4.block_scale.scale_vec::4X");
    }
#undef KB_MMA4
}
// 512 bytes of scales (32 lanes x 16 bytes) -> four TMEM columns of all four lane quarters; in order with the products of the same thread
template <bool PAIR>
__device__ __forceinline__ void tc_copy_scales(uint32_t tmem, uint64_t desc) {
    if constexpr (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// descriptor of such a piece: no swizzle, eight rows of 16 bytes contiguous, the next eight 128 bytes on
__device__ __forceinline__ uint64_t smem_desc_scales(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3ffffu) >> 4) | ((uint64_t)(128 >> 4) << 32) | (1ull << 46);
}

__device__ __forceinline__ void gemm4_tile(int w, const Gemm4Params& p, int& tm, int& tn) {   // as gemm_tile
    const int per_group = G_GROUP_M * p.tiles_n;
    const int first = (w / per_group) * G_GROUP_M, gsz = min(p.tiles_m - first, G_GROUP_M), in_g = w % per_group;
    tm = first + in_g % gsz;
    tn = in_g / gsz;
}

// v Phi(v) on a packed pair, in the form of gemm_sm100.cuh: with a = -min(|v|, 7), erfc(|v| / sqrt 2) = 2^(a Q(-a)) and v Phi(v) = max(v, 0) + a 2^(a Q(-a) - 1); max
// keeps a NaN. Here GELU is what bounds the epilogue, so Q has degree 7 and not 10: fitted to -log2(erfc(x / sqrt 2)) / x on [0, 7] (2000 Chebyshev nodes, least squares
// reweighted by the error of erfc times sqrt(erfc) + 1e-3). Largest error against float64 in fp32 2.4e-7, as with degree 10, relative 8e-6 within |v| < 3 and 6e-4 where
// the value is below 1e-5.
__device__ __forceinline__ uint64_t gelu2(uint64_t v) {
    float v0, v1;
    unpack2(v, v0, v1);
    const uint64_t a = pack2(fmaxf(-fabsf(v0), -7.f), fmaxf(-fabsf(v1), -7.f));
    auto both = [](float c) { return pack2(c, c); };
    uint64_t q = both(-3.179015664045437e-07f);
    q = fma2(q, a, both(-5.414401130110491e-06f));
    q = fma2(q, a, both(-3.436955466895597e-06f));
    q = fma2(q, a, both(0.0006369439070113003f));
    q = fma2(q, a, both(0.007798188831657171f));
    q = fma2(q, a, both(0.053058017045259476f));
    q = fma2(q, a, both(-0.4590109884738922f));
    q = fma2(q, a, both(1.151127815246582f));
    float t0, t1;
    unpack2(fma2(q, a, both(-1.f)), t0, t1);
    return fma2(a, pack2(ex2(t0), ex2(t1)), pack2(max0_nan(v0), max0_nan(v1)));
}

// Codes and scales of 32 neighbouring columns of a row (two blocks of NV4, one of MX4), packed pairs: 16 bytes, and the scale bytes from bit 0 on
template <int FMT>
__device__ __forceinline__ void quant32(const uint64_t* v, uint4& codes, uint32_t& scale_bytes) {
    uint32_t words[4];
    scale_bytes = 0u;
    constexpr int BLK = q4_block(FMT);
#pragma unroll
    for (int b = 0; b < 32 / BLK; b++) {
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < BLK / 2; e++) {
            float x, y;
            unpack2(v[b * BLK / 2 + e], x, y);
            top = max3_abs_nan(top, x, y);
        }
        const BlockScale<FMT> bs(__float_as_uint(top) & 0x7fffffffu, 1.f, 1.f);
        scale_bytes |= bs.byte << (8 * b);
#pragma unroll
        for (int i = 0; i < BLK / 8; i++) words[b * (BLK / 8) + i] = bs.codes(v + b * BLK / 2 + 4 * i);
    }
    codes = make_uint4(words[0], words[1], words[2], words[3]);
}

template <int EPI, int FMT, bool PAIR>
__global__ void __launch_bounds__(G4_THREADS, 1)
gemm4_kernel(const __grid_constant__ Gemm4Maps maps, const Gemm4Params p) {
    constexpr int BN = PAIR ? 256 : 128, TILE_M = PAIR ? 256 : 128;
    constexpr int BUF_COLS = 128, ACC_SF = BUF_COLS + BN;                 // TMEM: the second accumulator begins at BUF_COLS, the scales behind it
    constexpr int PIECES = FMT == FMT_MX4 ? 2 : 4;                        // scale pieces of a k step per row block
    constexpr int W_BLOCKS = PAIR ? 2 : 1;                                // row blocks of W whose scales a CTA holds
    constexpr int SF_COLS = 4 * PIECES * (1 + W_BLOCKS);                  // TMEM columns of a step's scales
    constexpr int SF_BUFS = PAIR && FMT == FMT_NV4 ? 2 : 4;               // steps of them in flight
    static_assert(ACC_SF + SF_BUFS * SF_COLS <= (int)TMEM_ALL_COLUMNS, "TMEM");
    constexpr uint32_t STAGE_TX = 32768 + PIECES * 512 * (1 + W_BLOCKS);
    constexpr bool OUT32 = EPI == EPI_F32 || EPI == EPI_RESID;
    constexpr int CW = 32, NCH = BN / CW;                                 // columns per chunk of the epilogue, which a warp has NCH / 4 of
    constexpr int BOX_COLS = OUT32 ? 16 : CW, BOXES = CW / BOX_COLS;      // a chunk leaves as one or two boxes of 32 rows x 64 bytes

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* const smem = smem_raw + (base - raw);
    uint8_t* const stage_out = smem + G4_STAGES * G4_STAGE_BYTES;
    uint8_t* const ctrl = stage_out + G4_EPI_WARPS * G4_STAGING_WARP;
    const uint32_t bars = smem_u32(ctrl);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(ctrl + 512);
    volatile uint32_t* const abort_flag = reinterpret_cast<volatile uint32_t*>(ctrl + 516);
    auto bar = [&](int i) { return bars + 8u * (uint32_t)i; };

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = PAIR ? cluster_ctarank() : 0u;                  // 0 issues the MMAs
    const int group = (int)blockIdx.x / (PAIR ? 2 : 1), n_groups = (int)gridDim.x / (PAIR ? 2 : 1);
    const int n_tiles = p.tiles_m * p.tiles_n, ksteps = (p.K + G4_K - 1) / G4_K;

    if (tid == 0) {
        for (int i = 0; i < G4BAR_COUNT; i++) mbar_init(bar(i), i >= G4BAR_ACC_EMPTY ? (PAIR ? 2u : 1u) * G4_EPI_WARPS : 1u);   // acc_empty: one arrival per epilogue warp of the group
        *abort_flag = 0u;
        mbar_fence_init();
        fence_proxy_async_smem();
    }
    if (warp == G4_EPI_WARPS + 1 && lane == 0) { tma_prefetch_desc(&maps.a); tma_prefetch_desc(&maps.w); tma_prefetch_desc(&maps.sa); tma_prefetch_desc(&maps.sw); }
    if (warp == G4_EPI_WARPS) {
        tmem_alloc(smem_u32(tmem_slot), TMEM_ALL_COLUMNS);
        tmem_relinquish();
    }
    pdl_launch();
    tc_fence_before();
    if (PAIR) { cluster_arrive(); cluster_wait(); } else __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem_base = 0u;                                    // see TMEM_ALL_COLUMNS
    pdl_wait();

    if (warp < G4_EPI_WARPS) {
        setmaxnreg_inc<104>();
        const int quarter = warp & 3, part = warp >> 2;                   // TMEM lanes [32 quarter, +32); every fourth chunk of columns
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        uint8_t* const my_stage = stage_out + warp * G4_STAGING_WARP;
        uint32_t use[2] = {0, 0};
        int k = 0;
        for (int w = group; w < n_tiles; w += n_groups, ++k) {
            const int buf = k & 1;
            int tm, tn;
            gemm4_tile(w, p, tm, tn);
            const int m0 = tm * TILE_M + (int)rank * GB_M, n0 = tn * BN;
            const bool ok = __all_sync(0xffffffffu, mbar_wait(bar(G4BAR_ACC_FULL + buf), use[buf] & 1u, abort_flag));
            ++use[buf];
            if (!ok) break;
            tc_fence_after();
            const int row = m0 + quarter * 32 + lane, nrow = p.M - (m0 + quarter * 32);
            // PAIR: the columns that both accumulators own first; the other chunk's load is under way while the first one is worked on
            uint32_t acc[NCH / 4][32];
            auto column = [&](int i) { return (part + 4 * (PAIR ? i ^ buf ^ 1 : i)) * CW; };
            tmem_ld32(tmem_base + lane_base + (uint32_t)(buf * BUF_COLS + column(0)), acc[0]);
            tmem_wait_ld();
            reg_fence32(acc[0]);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {                                              // what the next tile's products overwrite is in registers
                const uint32_t b = bar(G4BAR_ACC_EMPTY + (PAIR ? 0 : buf));
                if (PAIR && rank != 0) mbar_arrive_cluster_relaxed(mapa_u32(b, 0));
                else mbar_arrive(b);
            }
            if constexpr (PAIR) tmem_ld32(tmem_base + lane_base + (uint32_t)(buf * BUF_COLS + column(1)), acc[NCH / 4 - 1]);
#pragma unroll
            for (int i = 0; i < NCH / 4; i++) {
                if (i == 1) {
                    tmem_wait_ld();
                    reg_fence32(acc[NCH / 4 - 1]);
                }
                uint64_t v[CW / 2];
                const uint64_t alpha = pack2(p.alpha, p.alpha);
#pragma unroll
                for (int e = 0; e < 16; e++) v[e] = mul2(pack2u(acc[i][2 * e], acc[i][2 * e + 1]), alpha);
                const int c0 = n0 + column(i);
                if constexpr (EPI == EPI_GELU16 || EPI == EPI_GELU4) {
#pragma unroll
                    for (int c = 0; c < CW / 2; c++) v[c] = gelu2(v[c]);
                }
                if constexpr (EPI == EPI_GELU4) {
                    if (c0 + CW > p.N) {                                  // nothing of W's rows behind the last, whose scales may be anything
#pragma unroll
                        for (int c = 0; c < CW / 2; c++) {
                            float x, y;
                            unpack2(v[c], x, y);
                            v[c] = pack2(c0 + 2 * c < p.N ? x : 0.f, c0 + 2 * c + 1 < p.N ? y : 0.f);
                        }
                    }
                    // A thread has whole blocks: 16 bytes of codes and the scales of 32 columns at a time, stored as they are. The scales of a piece's blocks
                    // behind the last column are zeros: whoever has the last column writes them.
                    constexpr int PER = 32 / q4_block(FMT), PIECE = 4 * q4_block(FMT);
#pragma unroll
                    for (int q = 0; q < CW / 32; q++) {
                        const int c = c0 + 32 * q;
                        uint4 codes;
                        uint32_t sb;
                        quant32<FMT>(v + 16 * q, codes, sb);
                        if (row >= p.M || c >= p.N) continue;
                        *reinterpret_cast<uint4*>(p.codes + (size_t)row * p.ld_codes + (c >> 1)) = codes;
                        uint8_t* const s = p.scales + q4_scale_at(row, c / PIECE, p.pieces);
                        const int b = c % PIECE / q4_block(FMT);          // its first block in the piece
                        if (c + 32 >= p.N) {
                            const int blocks = (p.N - c + q4_block(FMT) - 1) / q4_block(FMT);
                            if (blocks < PER) sb &= 0xffu;
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                if (b + e < 4) s[b + e] = (uint8_t)(sb >> (8 * e));
                        } else if (PER == 2) {
                            *reinterpret_cast<uint16_t*>(s + b) = (uint16_t)sb;
                        } else {
                            s[b] = (uint8_t)sb;
                        }
                    }
                } else {
                    if constexpr (EPI == EPI_RESID) {
                        if (p.gate) {
#pragma unroll
                            for (int c = 0; c < CW / 2; c++)
                                v[c] = mul2(v[c], pack2(c0 + 2 * c < p.N ? p.gate[c0 + 2 * c] : 0.f, c0 + 2 * c + 1 < p.N ? p.gate[c0 + 2 * c + 1] : 0.f));
                        }
                    }
                    // 32 rows of the chunk as swizzled boxes in shared memory, which leave by TMA
#pragma unroll
                    for (int b = 0; b < BOXES; b++) {
                        const int x = c0 + b * BOX_COLS, y = m0 + quarter * 32;
                        if ((p.N & (OUT32 ? 3 : 7)) && x < p.N && x + BOX_COLS > p.N) {
                            // A box is cut at 16 bytes and not at the last column: where that lies inside 16 bytes, plain stores
                            if (row < p.M) {
#pragma unroll
                                for (int c = 0; c < BOX_COLS; c++) {
                                    if (x + c >= p.N) continue;
                                    float lo, hi;
                                    unpack2(v[(b * BOX_COLS + c) / 2], lo, hi);
                                    const float u = c & 1 ? hi : lo;
                                    const size_t at = (size_t)row * p.ldc + x + c;
                                    if constexpr (EPI == EPI_RESID) static_cast<float*>(p.C)[at] += u;
                                    else if constexpr (OUT32) static_cast<float*>(p.C)[at] = u;
                                    else static_cast<__half*>(p.C)[at] = __float2half_rn(u);
                                }
                            }
                            continue;
                        }
                        if (lane == 0) tma_store_wait_read();             // the box that was here has been read
                        __syncwarp();
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            uint4 pk;
                            if constexpr (OUT32) {
                                const uint64_t* const u = v + b * 8 + 2 * c;
                                pk = make_uint4((uint32_t)u[0], (uint32_t)(u[0] >> 32), (uint32_t)u[1], (uint32_t)(u[1] >> 32));
                            } else {
                                const uint64_t* const u = v + 4 * c;
                                auto two = [](uint64_t w) { float lo, hi; unpack2(w, lo, hi); return pack16<DT_F16>(lo, hi); };
                                pk = make_uint4(two(u[0]), two(u[1]), two(u[2]), two(u[3]));
                            }
                            *reinterpret_cast<uint4*>(my_stage + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)) = pk;
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0 && nrow > 0 && x < p.N) {
                            if constexpr (EPI == EPI_RESID) tma_reduce_add_3d(&maps.c, smem_u32(my_stage), x, y, 0);
                            else tma_store_3d(&maps.c, smem_u32(my_stage), x, y, 0);
                            tma_store_commit();
                        }
                    }
                }
            }
        }
        if (lane == 0) tma_store_wait_read();
    } else if (warp == G4_EPI_WARPS) {
        setmaxnreg_dec<56>();
        if (rank == 0 && elect_one()) {
            // the products of a step take the pipe 0.3 us, little more than what this thread spends on one: counters instead of remainders
            uint32_t st = 0, phase = 0;                                   // stage and its parity
            uint32_t old_st = G4_STAGES - SF_BUFS, old_phase = 1;         // those of the step that had this buffer of scales (passes at once where there was none)
            uint32_t sf = 0, use[2] = {0, 0};
            bool good = true;
            int k = 0;
            for (int w = group; w < n_tiles && good; w += n_groups, ++k) {
                const int buf = k & 1;
                const uint32_t acc = tmem_base + (uint32_t)(buf * BUF_COLS);
                if (PAIR) {
                    // the tile before this one is out of the shared columns, so the one before that is out of all of its own
                    if (k > 0) good = mbar_wait(bar(G4BAR_ACC_EMPTY), (uint32_t)(k - 1) & 1u, abort_flag);
                } else {
                    good = mbar_wait(bar(G4BAR_ACC_EMPTY + buf), (use[buf] & 1u) ^ 1u, abort_flag);   // passes at once for the first two tiles
                }
                ++use[buf];
                if (!good) break;
                tc_fence_after();
                for (int ks = 0; ks < ksteps; ++ks) {
                    good = mbar_wait(bar(G4BAR_FULL + st), phase, abort_flag);
                    // the products that read this buffer of scales are done
                    good = good && mbar_wait(bar(G4BAR_EMPTY + old_st), old_phase, abort_flag);
                    if (!good) break;
                    tc_fence_after();
                    const uint32_t a_s = base + st * G4_STAGE_BYTES;
                    const uint32_t sfa = tmem_base + ACC_SF + sf * SF_COLS, sfb = sfa + 4 * PIECES;
                    const uint64_t sdesc = smem_desc_scales(a_s + G4_SF_OFF);
#pragma unroll
                    for (int q = 0; q < PIECES; q++) {
                        tc_copy_scales<PAIR>(sfa + 4 * q, sdesc + (uint64_t)(q * 32));
#pragma unroll
                        for (int b = 0; b < W_BLOCKS; b++) tc_copy_scales<PAIR>(sfb + 4 * (q * W_BLOCKS + b), sdesc + (uint64_t)((PIECES * (1 + b) + q) * 32));
                    }
                    const uint64_t adesc = smem_desc_sw128(a_s, 16, 1024), wdesc = smem_desc_sw128(a_s + 16384, 16, 1024);
#pragma unroll
                    for (int kk = 0; kk < 4; kk++) {
                        const int q = kk * PIECES / 4, byte = FMT == FMT_MX4 ? (kk & 1) * 2 : 0;
                        mma_f4<FMT, PAIR>(acc, adesc + (uint64_t)(kk * 2), wdesc + (uint64_t)(kk * 2), idesc_f4(FMT == FMT_MX4, TILE_M, BN, byte), sfa + 4 * q,
                                          sfb + 4 * q * W_BLOCKS, (ks > 0 || kk > 0) ? 1u : 0u);
                    }
                    if (PAIR) tc_commit_pair(bar(G4BAR_EMPTY + st), (uint16_t)3); else tc_commit(bar(G4BAR_EMPTY + st));
                    if (++st == G4_STAGES) { st = 0; phase ^= 1u; }
                    if (++old_st == G4_STAGES) { old_st = 0; old_phase ^= 1u; }
                    if (++sf == SF_BUFS) sf = 0;
                }
                if (good) { if (PAIR) tc_commit_pair(bar(G4BAR_ACC_FULL + buf), (uint16_t)3); else tc_commit(bar(G4BAR_ACC_FULL + buf)); }
            }
        }
        __syncwarp();
    } else {
        setmaxnreg_dec<56>();
        if (warp == G4_EPI_WARPS + 1 && elect_one()) {
            uint32_t ring = 0;
            bool good = true;
            for (int w = group; w < n_tiles && good; w += n_groups) {
                int tm, tn;
                gemm4_tile(w, p, tm, tn);
                for (int ks = 0; ks < ksteps && good; ++ks, ++ring) {
                    const uint32_t st = ring % G4_STAGES;
                    good = mbar_wait(bar(G4BAR_EMPTY + st), ((ring / G4_STAGES) & 1u) ^ 1u, abort_flag);
                    if (!good) break;
                    const uint32_t a_s = base + st * G4_STAGE_BYTES, s_s = a_s + G4_SF_OFF;
                    if (PAIR) {
                        // both CTAs' bytes complete on the issuing CTA's barrier
                        if (rank == 0) mbar_expect_tx(bar(G4BAR_FULL + st), 2 * STAGE_TX);
                        const uint32_t fb = mapa_u32(bar(G4BAR_FULL + st), 0);
                        tma_load_3d_pair(a_s, &maps.a, fb, ks * 128, tm * TILE_M + (int)rank * 128, 0);
                        tma_load_3d_pair(a_s + 16384, &maps.w, fb, ks * 128, tn * BN + (int)rank * 128, 0);
                        tma_load_3d_pair(s_s, &maps.sa, fb, 0, ks * PIECES, tm * 2 + (int)rank);
#pragma unroll
                        for (int b = 0; b < W_BLOCKS; b++) tma_load_3d_pair(s_s + PIECES * 512 * (1 + b), &maps.sw, fb, 0, ks * PIECES, tn * W_BLOCKS + b);
                    } else {
                        const uint32_t fb = bar(G4BAR_FULL + st);
                        mbar_expect_tx(fb, STAGE_TX);
                        tma_load_3d(a_s, &maps.a, fb, ks * 128, tm * TILE_M, 0);
                        tma_load_3d(a_s + 16384, &maps.w, fb, ks * 128, tn * BN, 0);
                        tma_load_3d(s_s, &maps.sa, fb, 0, ks * PIECES, tm);
                        tma_load_3d(s_s + PIECES * 512, &maps.sw, fb, 0, ks * PIECES, tn);
                    }
                }
            }
            if (!good || *abort_flag) {
                // let the copies already requested land before the memory goes away, as in gemm16_kernel
                if (!PAIR || rank == 0) {
                    for (uint32_t k = ring > (uint32_t)G4_STAGES ? ring - G4_STAGES : 0u; k < ring; ++k) drain_wait(bar(G4BAR_FULL + k % G4_STAGES), (k / G4_STAGES) & 1u);
                } else {
                    const uint64_t t0 = globaltimer_ns();
                    while (globaltimer_ns() - t0 < 20000ull) {}
                }
            }
        }
        __syncwarp();
    }
    tc_fence_before();
    if (PAIR) { cluster_arrive(); cluster_wait(); } else __syncthreads();
    if (warp == G4_EPI_WARPS) {
        if (lane == 0 && *abort_flag) atomicOr(p.status, ST_TIMEOUT);
        tc_fence_after();
        tmem_dealloc(tmem_base, TMEM_ALL_COLUMNS);
    }
}

}  // namespace kb
