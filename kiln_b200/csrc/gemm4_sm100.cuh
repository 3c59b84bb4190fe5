// Product of two matrices of block-scaled 4-bit numbers (quant4.cuh) on sm_100a: C = epilogue(alpha * A[M,K] * W[N,K]^T). The tensor cores take the
// codes and the scales as they lie in memory: tcgen05.mma kind::mxf4 (MX4, a scale per 32) and kind::mxf4nvf4 (NV4, a scale per 16) multiply
// the 64 products of a k step by their blocks' scales and sum in fp32 in TMEM. Every product and its scaling is exact; only the sums round.
//
// The schedule is that of the fp16 product next door (gemm_sm100.cuh): persistent CTAs, one warp loads by TMA, one issues, eight run the epilogue of one
// tile under the main loop of the next. What differs: a k step in shared memory holds 256 columns (128 bytes) of each operand, plus their scales
// (2 KB per 128 rows for NV4, 1 KB for MX4), which tcgen05.cp copies to TMEM in front of the step's products, four lanes' quarters at a time.
//
// Two shapes. Single: one CTA per 128 x 128 tile. PAIR: two CTAs share a 256 x 256 tile (cta_group::2), each with its 128 rows of A, half of the W rows,
// the scales of its rows and of ALL 256 columns, and its 128 x 256 half of the accumulator. Two such accumulators fill TMEM and leave no room for
// scales, so they overlap: the first lies in columns [0, 256), the second in [128, 384), the scales behind them. The epilogue drains the 128 columns that
// both own first, and then the next tile's products may begin: half of the epilogue still runs under them.
#pragma once
#include "gemm_sm100.cuh"   // gelu, elect_one, pack16
#include "quant4.cuh"

namespace kb {

constexpr int EPI_GELU4 = 5;                               // C leaves in 4 bits: codes and scales of gelu(alpha * acc)

constexpr int G4_K = 256;                                  // columns of a k step: 128 bytes of codes
constexpr int G4_STAGES = 5;
constexpr int G4_SF_OFF = 32768;                           // scales of a stage: A's 128 rows, then W's
constexpr int G4_STAGE_BYTES = G4_SF_OFF + 6144;
constexpr int G4_STAGING_WARP = 4096;
constexpr int G4_SMEM = G4_STAGES * G4_STAGE_BYTES + G_EPI_WARPS * G4_STAGING_WARP + 1024 + 1024;
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

// Codes and scales of 32 neighbouring columns of a row (two blocks of NV4, one of MX4): 16 bytes, and the scale bytes from bit 0 on
template <int FMT>
__device__ __forceinline__ void quant32(const float* v, uint4& codes, uint32_t& scale_bytes) {
    uint32_t words[4];
    scale_bytes = 0u;
    constexpr int BLK = q4_block(FMT);
#pragma unroll
    for (int b = 0; b < 32 / BLK; b++) {
        uint32_t top = 0u;
#pragma unroll
        for (int e = 0; e < BLK; e++) top = max(top, __float_as_uint(v[b * BLK + e]) & 0x7fffffffu);
        const BlockScale<FMT> bs(top, 1.f);
        scale_bytes |= bs.byte << (8 * b);
#pragma unroll
        for (int i = 0; i < BLK / 8; i++) {
            float q[8];
#pragma unroll
            for (int e = 0; e < 8; e++) q[e] = bs(v[b * BLK + 8 * i + e], 1.f);
            words[b * (BLK / 8) + i] = e2m1_pack8(q);
        }
    }
    codes = make_uint4(words[0], words[1], words[2], words[3]);
}

template <int EPI, int FMT, bool PAIR>
__global__ void __launch_bounds__(G_THREADS, 1)
gemm4_kernel(const __grid_constant__ Gemm4Maps maps, const Gemm4Params p) {
    constexpr int BN = PAIR ? 256 : 128, TILE_M = PAIR ? 256 : 128;
    constexpr int BUF_COLS = 128, ACC_SF = BUF_COLS + BN;                 // TMEM: the second accumulator begins at BUF_COLS, the scales behind it
    constexpr int PIECES = FMT == FMT_MX4 ? 2 : 4;                        // scale pieces of a k step per row block
    constexpr int W_BLOCKS = BN / 128;                                    // row blocks of W whose scales a CTA holds
    constexpr int SF_COLS = 4 * PIECES * (1 + W_BLOCKS);                  // TMEM columns of a step's scales
    constexpr int SF_BUFS = PAIR && FMT == FMT_NV4 ? 2 : 4;               // steps of them in flight
    static_assert(ACC_SF + SF_BUFS * SF_COLS <= (int)TMEM_ALL_COLUMNS, "TMEM");
    constexpr uint32_t STAGE_TX = 32768 + PIECES * 512 * (1 + W_BLOCKS);
    constexpr bool OUT32 = EPI == EPI_F32 || EPI == EPI_RESID;
    constexpr int CW = 64, NCH = BN / CW, BOX_COLS = OUT32 ? 32 : 64, BOXES = CW / BOX_COLS;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* const smem = smem_raw + (base - raw);
    uint8_t* const stage_out = smem + G4_STAGES * G4_STAGE_BYTES;
    uint8_t* const ctrl = stage_out + G_EPI_WARPS * G4_STAGING_WARP;
    const uint32_t bars = smem_u32(ctrl);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(ctrl + 512);
    volatile uint32_t* const abort_flag = reinterpret_cast<volatile uint32_t*>(ctrl + 516);
    auto bar = [&](int i) { return bars + 8u * (uint32_t)i; };

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = PAIR ? cluster_ctarank() : 0u;                  // 0 issues the MMAs
    const int group = (int)blockIdx.x / (PAIR ? 2 : 1), n_groups = (int)gridDim.x / (PAIR ? 2 : 1);
    const int n_tiles = p.tiles_m * p.tiles_n, ksteps = (p.K + G4_K - 1) / G4_K;

    if (tid == 0) {
        for (int i = 0; i < G4BAR_COUNT; i++) mbar_init(bar(i), i >= G4BAR_ACC_EMPTY ? (PAIR ? 2u : 1u) * G_EPI_WARPS : 1u);   // acc_empty: one arrival per epilogue warp of the group
        *abort_flag = 0u;
        mbar_fence_init();
        fence_proxy_async_smem();
    }
    if (warp == G_EPI_WARPS + 1 && lane == 0) { tma_prefetch_desc(&maps.a); tma_prefetch_desc(&maps.w); tma_prefetch_desc(&maps.sa); tma_prefetch_desc(&maps.sw); }
    if (warp == G_EPI_WARPS) {
        tmem_alloc(smem_u32(tmem_slot), TMEM_ALL_COLUMNS);
        tmem_relinquish();
    }
    pdl_launch();
    tc_fence_before();
    if (PAIR) { cluster_arrive(); cluster_wait(); } else __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem_base = 0u;                                    // see TMEM_ALL_COLUMNS
    pdl_wait();

    if (warp < G_EPI_WARPS) {
        setmaxnreg_inc<224>();
        const int quarter = warp & 3, half = warp >> 2;                   // TMEM lanes [32 quarter, +32); every other chunk of columns
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
#pragma unroll 1
            for (int i = 0; i < NCH / 2; i++) {
                const int ch = half + 2 * (PAIR ? i ^ buf ^ 1 : i);       // PAIR: the columns that both accumulators own first
                float v[CW];
                {
                    uint32_t a[CW / 32][32];
#pragma unroll
                    for (int q = 0; q < CW / 32; q++) tmem_ld32(tmem_base + lane_base + (uint32_t)(buf * BUF_COLS + ch * CW + 32 * q), a[q]);
                    tmem_wait_ld();
#pragma unroll
                    for (int q = 0; q < CW / 32; q++) {
                        reg_fence32(a[q]);
#pragma unroll
                        for (int e = 0; e < 32; e++) v[32 * q + e] = __uint_as_float(a[q][e]) * p.alpha;
                    }
                }
                if (i == 0) {                                             // single: the only chunk; the next tile's products may come
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (PAIR && rank != 0) mbar_arrive_cluster(mapa_u32(bar(G4BAR_ACC_EMPTY), 0));
                        else mbar_arrive(bar(G4BAR_ACC_EMPTY + (PAIR ? 0 : buf)));
                    }
                }
                const int c0 = n0 + ch * CW;
                if constexpr (EPI == EPI_GELU16 || EPI == EPI_GELU4) {
#pragma unroll
                    for (int c = 0; c < CW; c++) v[c] = gelu(v[c]);
                }
                if constexpr (EPI == EPI_GELU4) {
                    if (c0 + CW > p.N) {                                  // nothing of W's rows behind the last, whose scales may be anything
#pragma unroll
                        for (int c = 0; c < CW; c++) v[c] = c0 + c < p.N ? v[c] : 0.f;
                    }
                    // a thread has whole blocks: 32 bytes of codes and the scales of 64 columns, stored as they are
                    uint4 codes[2];
                    uint32_t sb[2];
                    quant32<FMT>(v, codes[0], sb[0]);
                    quant32<FMT>(v + 32, codes[1], sb[1]);
                    if (row < p.M && c0 < p.N) {
                        uint8_t* const dst = p.codes + (size_t)row * p.ld_codes + (c0 >> 1);
                        *reinterpret_cast<uint4*>(dst) = codes[0];
                        if (c0 + 32 < p.N) *reinterpret_cast<uint4*>(dst + 16) = codes[1];
                        // scales of blocks behind the last column are zeros
                        constexpr int PER = 32 / q4_block(FMT);
                        uint32_t word = sb[0] | (c0 + 32 < p.N ? sb[1] << (8 * PER) : 0u);
                        const int blocks = (p.N - c0 + q4_block(FMT) - 1) / q4_block(FMT);
                        if (blocks < 2 * PER) word &= (1u << (8 * blocks)) - 1u;
                        if constexpr (FMT == FMT_NV4) {
                            *reinterpret_cast<uint32_t*>(p.scales + q4_scale_at(row, c0 >> 6, p.pieces)) = word;
                        } else {                                          // half a piece; behind the last column the other half as well
                            uint8_t* const s = p.scales + q4_scale_at(row, c0 >> 7, p.pieces);
                            if ((c0 & 64) == 0 && c0 + 64 >= p.N) *reinterpret_cast<uint32_t*>(s) = word;
                            else *reinterpret_cast<uint16_t*>(s + ((c0 >> 5) & 2)) = (uint16_t)word;
                        }
                    }
                } else {
                    if constexpr (EPI == EPI_RESID) {
                        if (p.gate) {
#pragma unroll
                            for (int c = 0; c < CW; c++) v[c] *= c0 + c < p.N ? p.gate[c0 + c] : 0.f;
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
                                    const size_t at = (size_t)row * p.ldc + x + c;
                                    if constexpr (EPI == EPI_RESID) static_cast<float*>(p.C)[at] += v[b * 32 + c];
                                    else if constexpr (OUT32) static_cast<float*>(p.C)[at] = v[b * 32 + c];
                                    else static_cast<__half*>(p.C)[at] = __float2half_rn(v[c]);
                                }
                            }
                            continue;
                        }
                        if (lane == 0) tma_store_wait_read();             // the box that was here has been read
                        __syncwarp();
#pragma unroll
                        for (int c = 0; c < 8; c++) {
                            uint4 pk;
                            if constexpr (OUT32) {
                                const float* const u = v + b * 32 + 4 * c;
                                pk = make_uint4(__float_as_uint(u[0]), __float_as_uint(u[1]), __float_as_uint(u[2]), __float_as_uint(u[3]));
                            } else {
                                const float* const u = v + 8 * c;
                                pk.x = pack16<DT_F16>(u[0], u[1]); pk.y = pack16<DT_F16>(u[2], u[3]);
                                pk.z = pack16<DT_F16>(u[4], u[5]); pk.w = pack16<DT_F16>(u[6], u[7]);
                            }
                            *reinterpret_cast<uint4*>(my_stage + lane * 128 + ((c ^ (lane & 7)) << 4)) = pk;
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
    } else if (warp == G_EPI_WARPS) {
        setmaxnreg_dec<56>();
        if (rank == 0 && elect_one()) {
            uint32_t ring = 0, use[2] = {0, 0};
            bool good = true;
            int k = 0;
            for (int w = group; w < n_tiles && good; w += n_groups, ++k) {
                const int buf = k & 1;
                if (PAIR) {
                    // the tile before this one is out of the shared columns, so the one before that is out of all of its own
                    if (k > 0) good = mbar_wait(bar(G4BAR_ACC_EMPTY), (uint32_t)(k - 1) & 1u, abort_flag);
                } else {
                    good = mbar_wait(bar(G4BAR_ACC_EMPTY + buf), (use[buf] & 1u) ^ 1u, abort_flag);   // passes at once for the first two tiles
                }
                ++use[buf];
                if (!good) break;
                tc_fence_after();
                for (int ks = 0; ks < ksteps && good; ++ks, ++ring) {
                    const uint32_t st = ring % G4_STAGES;
                    good = mbar_wait(bar(G4BAR_FULL + st), (ring / G4_STAGES) & 1u, abort_flag);
                    // the products that read this buffer of scales are done
                    if (good && ring >= SF_BUFS) good = mbar_wait(bar(G4BAR_EMPTY + (ring - SF_BUFS) % G4_STAGES), ((ring - SF_BUFS) / G4_STAGES) & 1u, abort_flag);
                    if (!good) break;
                    tc_fence_after();
                    const uint32_t a_s = base + st * G4_STAGE_BYTES;
                    const uint32_t sfa = tmem_base + ACC_SF + (ring % SF_BUFS) * SF_COLS, sfb = sfa + 4 * PIECES;
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
                        mma_f4<FMT, PAIR>(tmem_base + (uint32_t)(buf * BUF_COLS), adesc + (uint64_t)(kk * 2), wdesc + (uint64_t)(kk * 2),
                                          idesc_f4(FMT == FMT_MX4, TILE_M, BN, byte), sfa + 4 * q, sfb + 4 * q * W_BLOCKS, (ks > 0 || kk > 0) ? 1u : 0u);
                    }
                    if (PAIR) tc_commit_pair(bar(G4BAR_EMPTY + st), (uint16_t)3); else tc_commit(bar(G4BAR_EMPTY + st));
                }
                if (good) { if (PAIR) tc_commit_pair(bar(G4BAR_ACC_FULL + buf), (uint16_t)3); else tc_commit(bar(G4BAR_ACC_FULL + buf)); }
            }
        }
        __syncwarp();
    } else {
        setmaxnreg_dec<56>();
        if (warp == G_EPI_WARPS + 1 && elect_one()) {
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
    if (warp == G_EPI_WARPS) {
        if (lane == 0 && *abort_flag) atomicOr(p.status, ST_TIMEOUT);
        tc_fence_after();
        tmem_dealloc(tmem_base, TMEM_ALL_COLUMNS);
    }
}

}  // namespace kb
