// Dropout whose mask is never stored: y = keep ? x S / (S - t) : 0, plus a residual if there is one, S = 65536, t = round(S p). The mask is a
// function of (seed, offset, row, column), so the gradient is the same call on the gradient of y: the 16-bit number of element (r, c) is half
// word c % 8 of Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) of
// counter (c / 8, r, offset) under key seed; kept where it is no less than t. 16 bits and not 32 per element halve the integer work, which at
// 32 bits would take longer than the memory; the scale goes by the rounded t, so the expectation is x exactly. A dropped element is
// a zero whatever it was (infinities and NaN too). seed and offset lie in device memory: a captured graph takes new ones at each replay.
#pragma once
#include "quant4.cuh"   // load8, store8

namespace kb {

// the keys of the ten rounds
struct PhiloxKeys {
    uint32_t a[10], b[10];
    __device__ __forceinline__ explicit PhiloxKeys(unsigned long long seed) {
#pragma unroll
        for (int i = 0; i < 10; i++) { a[i] = (uint32_t)seed + i * 0x9E3779B9u; b[i] = (uint32_t)(seed >> 32) + i * 0xBB67AE85u; }
    }
    // in registers from here on, not summed up again for every counter: a sixth of the instructions
    __device__ __forceinline__ void keep() {
#pragma unroll
        for (int i = 0; i < 10; i++) asm volatile("" : "+r"(a[i]), "+r"(b[i]));
    }
};
__device__ __forceinline__ uint4 philox4x32(uint4 c, const PhiloxKeys& k) {
#pragma unroll
    for (int i = 0; i < 10; i++) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c.x, p1 = (uint64_t)0xCD9E8D57u * c.z;
        c = make_uint4((uint32_t)(p1 >> 32) ^ c.y ^ k.a[i], (uint32_t)p1, (uint32_t)(p0 >> 32) ^ c.w ^ k.b[i], (uint32_t)p0);
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
};

// A thread keeps its eight columns and goes down the rows, the next row's load under the ten rounds of this one's. Of 16-bit numbers the integer work bounds
// it (113 instructions per eight elements; the issue slots 52 % busy, the warps waiting for the multiplier), and one round of thread blocks that keep the rounds' keys is
// best; of fp32 numbers the memory, and many short thread blocks keep more loads under way. Measured on B200, 4096 x 8192, a thread block per row -> one round: bf16 34.9
// -> 26.2 us (5.1 TB/s), with a residual 45.1 -> 35.3 (5.7); fp32 42.5 (6.3 TB/s) -> 57.8, so not taken there.
constexpr int DROP_THREADS_LOG2 = 8, DROP_THREADS = 1 << DROP_THREADS_LOG2;
template <typename InT, typename OutT> __host__ __device__ constexpr bool drop_one_round() { return sizeof(InT) == 2 && sizeof(OutT) == 2; }
// Thread blocks of one round, by the registers: 45 without a residual, 56 with one. (Compiled with a launch bound of 5 blocks, the kernel without a residual takes 31.4 us.)
template <bool RESID, bool WIDE> __host__ __device__ constexpr int drop_blocks_per_sm() { return (RESID ? 4 : 5) - !WIDE; }

// WIDE: every row of every matrix starts on 16 bytes. Else the lanes of a row (`width` of a warp's) read and write theirs across, see load_across.
template <typename InT, typename OutT, bool RESID, bool WIDE>
__global__ void __launch_bounds__(DROP_THREADS, !WIDE ? RESID ? 3 : 4 : drop_one_round<InT, OutT>() || RESID ? 4 : 6)
dropout_kernel(const DropoutParams p) {
    __shared__ Raw8<InT> tiles_x[WIDE ? 1 : DROP_THREADS];
    __shared__ Raw8<OutT> tiles_y[WIDE ? 1 : DROP_THREADS], tiles_r[WIDE || !RESID ? 1 : DROP_THREADS];
    pdl_launch();
    pdl_wait();
    const unsigned block_rows = DROP_THREADS >> p.width_log2, step = gridDim.x * block_rows;
    unsigned row = blockIdx.x * block_rows + (threadIdx.x >> p.width_log2);
    const int g = (int)(blockIdx.y << p.width_log2) + (int)(threadIdx.x & ((1u << p.width_log2) - 1u)), c = g * 8;
    const int width = min(32, 1 << p.width_log2), lane = threadIdx.x & (width - 1), first = c - 8 * lane;
    const unsigned place = threadIdx.x - lane;                         // of the lanes that share a row, the first
    const unsigned above = WIDE ? 0u : (threadIdx.x & 31u) >> p.width_log2;      // rows of the warp above this one's; the warp stays together for the first one's sake
    if (row - above >= (unsigned)p.rows || (WIDE ? c : first) >= p.cols) return;
    const int cols = WIDE || row < (unsigned)p.rows ? p.cols : 0;      // of a row behind the last nothing is read or written
    const InT* x = static_cast<const InT*>(p.x) + (size_t)row * p.ld_x;
    const OutT* res = static_cast<const OutT*>(p.resid) + (RESID ? (size_t)row * p.ld_r : 0);
    OutT* y = static_cast<OutT*>(p.y) + (size_t)row * p.ld_y;
    const size_t dx = (size_t)step * p.ld_x, dr = (size_t)step * p.ld_r, dy = (size_t)step * p.ld_y;
    auto load = [&](const auto* from, int n) { return WIDE ? load8_raw(from, c, n) : load_across(from, first, n, lane, width); };
    Raw8<InT> in = load(x, cols);
    Raw8<OutT> add;
    if (RESID) add = load(res, cols);
    const unsigned long long seed = p.rng[0], offset = p.rng[1];
    const uint32_t t = p.t << 16;
    PhiloxKeys keys(seed);
    if (drop_one_round<InT, OutT>()) keys.keep();
    int now = cols;
    while (true) {
        if (!WIDE) {
            if (RESID) add = across_to_own(add, tiles_r + place, lane, width);
            in = across_to_own(in, tiles_x + place, lane, width);
        }
        const F8 v = Io<InT>::f8(in);
        F8 out;
        if (RESID) out = Io<OutT>::f8(add);
        const unsigned next = row + step;
        const bool more = next > row && next - above < (unsigned)p.rows;       // (and not beyond 2^32)
        const int then = WIDE || next < (unsigned)p.rows ? p.cols : 0;
        if (more) {
            x += dx;
            in = load(x, then);
            if (RESID) { res += dr; add = load(res, then); }
        }
        const uint4 w = philox4x32(make_uint4((uint32_t)g, row, (uint32_t)offset, (uint32_t)(offset >> 32)), keys);
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 8; e++) {
            // a half word against t is the word, with that half on top, against 2^16 t
            const uint32_t r = (e & 1) ? words[e >> 1] : words[e >> 1] << 16;
            const float kept = r >= t ? __fmul_rn(v.v[e], p.scale) : 0.f;
            out.v[e] = RESID ? __fadd_rn(out.v[e], kept) : kept;       // product and sum rounded apart, with a residual and without
        }
        if (WIDE) {
            store8(y, c, p.cols, out);
        } else {
            Raw8<OutT> own;
            Io<OutT>::st8(reinterpret_cast<OutT*>(own.u), out);
            store_across(own, tiles_y + place, y, first, now, lane, width);
        }
        if (!more) break;
        y += dy;
        row = next;
        now = then;
    }
}

}  // namespace kb
