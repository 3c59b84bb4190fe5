// The 4-bit product for a single token: C[n] = epilogue(alpha * sum_k A[k] W[n,k]) by the ordinary cores. A tile of the tensor cores would be empty but for one
// row of 128, and with few tiles most SMs would be idle; here all of them stream their share of W, N K (1/2 + 1/block) bytes.
//
// A warp takes four rows of W that are 32 apart (their scales lie side by side in one 16-byte word of a piece), a lane 32 columns at a time, the next 32 on
// their way. The codes of both sides become fp16 (each value is one of its numbers) and are multiplied in pairs there: the products are multiples of 1/4
// up to 36 and a block of 16 gives each half of a pair eight of them, multiples of 1/4 up to 288, which eleven bits hold exactly. So a block's sum is exact; it
// is scaled and summed over the blocks in fp32. What bounds it is latency: with N 8192, K 2048 a lane has two pieces of 32 columns, the issue slots are 42 % busy and memory is at 16 %.
// Measured on B200, device time, tensor cores -> this: N 2048, K 2048, NV4 4.3 -> 2.5 us, N 8192 5.6 -> 3.8, MX4 5.4 -> 4.0, N 2048, K 8192 9.1 -> 6.2, 8192 x 8192 18.8 -> 11.8.
// (Two tokens in this form: as long as the tensor cores take for up to 128.)
#pragma once
#include "gemm4_sm100.cuh"   // gelu2
#include "quant4.cuh"

namespace kb {

constexpr int GV4_WARPS = 4, GV4_ROWS = 4;                  // rows of W of a warp

struct Gemv4Params {
    const uint8_t *a, *a_scales, *w, *w_scales;
    void* C;
    const float* gate;
    int N, K, ldw, pieces;                                  // K: columns, in memory padded to 32 with zeros; pieces of a row block, of both sides
    float alpha;
    int epi;
};

// a lane's 32 columns of A and of four rows of W, and the words that hold their scales
struct Gemv4Chunk {
    uint4 a, w[GV4_ROWS], sw;
    uint32_t sa;
};

// the scales of the 16-column halves of a lane's 32 columns, from the word that holds the four blocks of its piece
template <int FMT>
__device__ __forceinline__ float2 gv4_scales(uint32_t word, int chunk) {
    if (FMT == FMT_NV4) {
        const uint32_t two = (chunk & 1) ? word >> 16 : word;
        return make_float2(e4m3_value(two & 0xffu), e4m3_value((two >> 8) & 0xffu));
    }
    const float s = q4_scale_value<FMT_MX4>((word >> (8 * (chunk & 3))) & 0xffu);
    return make_float2(s, s);
}
__device__ __forceinline__ __half2 gv4_h2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }

// acc + sa sw sum for MX4. The product of two scales may leave fp32 where the term does not (the block's sum may be 0): scales on the same side of 1 are therefore
// multiplied with one after the other, so that what overflows or vanishes on the way does so in the term as well. (NV4's products lie in 2^-18 ... 2^18.)
__device__ __forceinline__ float gv4_add_mx4(float sa, float sw, float sum, float acc) {
    const bool apart = (sa < 1.f) == (sw < 1.f);
    return fmaf(apart ? sw : sa * sw, apart ? sum * sa : sum, acc);
}

template <int FMT>
__global__ void __launch_bounds__(32 * GV4_WARPS)
gemv4_kernel(const Gemv4Params p) {
    pdl_launch();
    pdl_wait();
    const int lane = threadIdx.x & 31, group = (int)blockIdx.x * GV4_WARPS + (int)(threadIdx.x >> 5);   // 32 groups of four rows to a row block
    const int n0 = (group >> 5) * 128 + (group & 31);
    if (n0 >= p.N) return;
    const int chunks = (p.K + 31) / 32;
    constexpr int PER_PIECE = FMT == FMT_NV4 ? 2 : 4;       // chunks of a piece of scales
    const uint8_t* const ws = p.w_scales + (size_t)(group >> 5) * p.pieces * 512 + (group & 31) * 16;
    const int real = min(GV4_ROWS, (p.N - n0 + 31) / 32);   // rows that exist
    auto load = [&](int c) {
        Gemv4Chunk k;
#pragma unroll
        for (int j = 0; j < GV4_ROWS; j++)
            k.w[j] = j < real ? __ldcg(reinterpret_cast<const uint4*>(p.w + (size_t)(n0 + 32 * j) * p.ldw) + c) : make_uint4(0u, 0u, 0u, 0u);
        k.sw = __ldcg(reinterpret_cast<const uint4*>(ws + (size_t)(c / PER_PIECE) * 512));
        k.a = *(reinterpret_cast<const uint4*>(p.a) + c);
        k.sa = *reinterpret_cast<const uint32_t*>(p.a_scales + (size_t)(c / PER_PIECE) * 512);
        return k;
    };
    float acc[GV4_ROWS] = {0.f, 0.f, 0.f, 0.f};
    Gemv4Chunk next;
    if (lane < chunks) next = load(lane);
    for (int c = lane; c < chunks; c += 32) {
        const Gemv4Chunk k = next;
        if (c + 32 < chunks) next = load(c + 32);
        const uint32_t sws[GV4_ROWS] = {k.sw.x, k.sw.y, k.sw.z, k.sw.w};
        const float2 fa = gv4_scales<FMT>(k.sa, c);
        float half[GV4_ROWS];                               // MX4: the first half of the block
#pragma unroll
        for (int b = 0; b < 2; b++) {                       // 16 columns at a time: 8 bytes of codes
            uint32_t a[8];
            e2m1_unpack8(b ? k.a.z : k.a.x, *reinterpret_cast<uint32_t(*)[4]>(a));
            e2m1_unpack8(b ? k.a.w : k.a.y, *reinterpret_cast<uint32_t(*)[4]>(a + 4));
#pragma unroll
            for (int j = 0; j < GV4_ROWS; j++) {
                uint32_t w[8];
                e2m1_unpack8(b ? k.w[j].z : k.w[j].x, *reinterpret_cast<uint32_t(*)[4]>(w));
                e2m1_unpack8(b ? k.w[j].w : k.w[j].y, *reinterpret_cast<uint32_t(*)[4]>(w + 4));
                __half2 s = __hmul2(gv4_h2(a[0]), gv4_h2(w[0]));
#pragma unroll
                for (int i = 1; i < 8; i++) s = __hfma2(gv4_h2(a[i]), gv4_h2(w[i]), s);
                const float2 f = __half22float2(s), fw = gv4_scales<FMT>(sws[j], c);
                // exact but for the sum: 8 bits of scales, 12 of the block (MX4: 13). Rows that do not exist may have scales of anything
                if (FMT == FMT_NV4) { if (j < real) acc[j] = fmaf((b ? fa.y : fa.x) * (b ? fw.y : fw.x), f.x + f.y, acc[j]); }
                else if (b == 0) half[j] = f.x + f.y;
                else if (j < real) acc[j] = gv4_add_mx4(fa.x, fw.x, half[j] + (f.x + f.y), acc[j]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < GV4_ROWS; j++)
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], d);
    const int n = n0 + 32 * lane;                           // lane j stores row j
    if (lane >= real) return;
    const float v = (lane == 0 ? acc[0] : lane == 1 ? acc[1] : lane == 2 ? acc[2] : acc[3]) * p.alpha;
    if (p.epi == EPI_F32) static_cast<float*>(p.C)[n] = v;
    else if (p.epi == EPI_RESID) static_cast<float*>(p.C)[n] += p.gate ? p.gate[n] * v : v;
    else {
        float g, same;
        unpack2(gelu2(pack2(v, v)), g, same);                  // the GELU of the form for several rows
        static_cast<__half*>(p.C)[n] = __float2half_rn(p.epi == EPI_GELU16 ? g : v);
    }
}

}  // namespace kb
