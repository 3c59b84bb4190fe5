// Dropout whose mask is never stored: y = keep ? x S / (S - t) : 0, plus a residual if there is one, S = 65536, t = round(S p). The mask is a
// function of (seed, offset, row, column), so the gradient is the same call on the gradient of y: the 16-bit number of element (r, c) is half
// word c % 8 of Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) of
// counter (c / 8, r, offset) under key seed; kept where it is no less than t. 16 bits and not 32 per element halve the integer work, which at
// 32 bits would take longer than the memory; the scale goes by the rounded t, so the expectation is x exactly. A dropped element is
// a zero whatever it was (infinities and NaN too). seed and offset lie in device memory: a captured graph takes new ones at each replay.
#pragma once
#include "quant4.cuh"   // load8, store8

namespace kb {

__device__ __forceinline__ uint4 philox4x32(uint4 c, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int i = 0; i < 10; i++) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c.x, p1 = (uint64_t)0xCD9E8D57u * c.z;
        c = make_uint4((uint32_t)(p1 >> 32) ^ c.y ^ k0, (uint32_t)p1, (uint32_t)(p0 >> 32) ^ c.w ^ k1, (uint32_t)p0);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return c;
}

struct DropoutParams {
    const void* x;
    const void* resid;                    // of the output's type, or null
    void* y;
    const unsigned long long* rng;        // seed, offset
    int rows, cols, ld_x, ld_r, ld_y;
    int width_log2;                       // threads of a block side by side on a row
    unsigned t;                           // a 16-bit number below t drops its element
    float scale;
    bool wide;                            // every row of every matrix starts on 16 bytes
};

// A thread takes DROP_GROUPS groups of eight columns, its loads first.
constexpr int DROP_THREADS_LOG2 = 8, DROP_THREADS = 1 << DROP_THREADS_LOG2, DROP_GROUPS = 1;

template <typename InT, typename OutT>
__global__ void __launch_bounds__(DROP_THREADS)
dropout_kernel(const DropoutParams p) {
    pdl_launch();
    pdl_wait();
    const int width = 1 << p.width_log2;
    const unsigned row = blockIdx.x * (unsigned)(DROP_THREADS >> p.width_log2) + (threadIdx.x >> p.width_log2);
    const int g0 = (int)blockIdx.y * (DROP_GROUPS * width) + (int)(threadIdx.x & (unsigned)(width - 1));
    if (row >= (unsigned)p.rows) return;
    const InT* const x = static_cast<const InT*>(p.x) + (size_t)row * p.ld_x;
    OutT* const y = static_cast<OutT*>(p.y) + (size_t)row * p.ld_y;
    const unsigned long long seed = p.rng[0], offset = p.rng[1];
    const uint32_t t = p.t << 16;
    F8 in[DROP_GROUPS], out[DROP_GROUPS];
#pragma unroll
    for (int i = 0; i < DROP_GROUPS; i++) {
        const int c = (g0 + i * width) * 8;
        if (c >= p.cols) break;
        in[i] = load8(x, c, p.cols, p.wide);
        if (p.resid) out[i] = load8(static_cast<const OutT*>(p.resid) + (size_t)row * p.ld_r, c, p.cols, p.wide);
        else
#pragma unroll
            for (int e = 0; e < 8; e++) out[i].v[e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < DROP_GROUPS; i++) {
        const int g = g0 + i * width, c = g * 8;
        if (c >= p.cols) break;
        const uint4 w = philox4x32(make_uint4((uint32_t)g, row, (uint32_t)offset, (uint32_t)(offset >> 32)), (uint32_t)seed, (uint32_t)(seed >> 32));
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 8; e++) {
            // a half word against t is the word, with that half on top, against 2^16 t
            const uint32_t r = (e & 1) ? words[e >> 1] : words[e >> 1] << 16;
            if (r >= t) out[i].v[e] = __fadd_rn(out[i].v[e], __fmul_rn(in[i].v[e], p.scale));   // product and sum rounded apart, with a residual and without
        }
        store8(y, c, p.cols, p.wide, out[i]);
    }
}

}  // namespace kb
