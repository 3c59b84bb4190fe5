// Rotary positions of up to four tensors (q and k, or their gradients) in one launch: of every head's first `rot` elements pair i turns by the
// angle t = pos[axis_i] f_i, (a, b) -> (a cos t - b sin t, b cos t + a sin t) * amplitude; the pairs are (i, i + rot / 2) (half) or
// (2 i, 2 i + 1) (interleaved), the rest of the head is copied. The inverse turns by -t: it is the gradient.
//
// The angle of a far position turns thousands of times, and fp32 has lost its fraction by then. Here a frequency is a 64-bit fraction of a turn
// and a position an integer, so their product modulo 2^64 IS the fraction of the turn, exactly, in two integer multiplications. What rounds is the
// fraction on its way into an fp32 number of half turns in [-1, 1): by 2^-25 of a half turn at most (9.4e-8 rad; the 32 bits cut off before are 2^-32 of a turn), then
// the sine and cosine themselves (2 units of fp32) and their product with the amplitude.
//
// Bound by memory. The sines of a row serve all of its heads of all tensors: a thread block takes a row or several (rope_split), fills shared memory
// with one (cos, sin) per pair while its first loads are under way, and every thread keeps those of its eight elements as it goes from head to head.
// Measured on B200, device time: q and k of 1536 rows, 16 heads of 128 each, half, fp32 10.3 us (4.9 TB/s), fp16 6.1; 4096 rows fp16 half 12.5 (5.4), interleaved 12.8; 8190 rows, 16 + 4
// heads, 96 of 128 interleaved, bf16 16.3 (5.1).
#pragma once
#include "quant4.cuh"   // to_f32, from_f32

namespace kb {

constexpr int ROPE_MAX_PAIRS = 128, ROPE_MAX_TENSORS = 4, ROPE_THREADS = 128;
constexpr int ROPE_SLOTS = 1024;                       // (row, pair) places in shared memory

struct RopeTensor {
    const void* x;
    void* y;
    int first, ld_x, ld_y;                             // first: its first head among those of all tensors
};
struct RopeParams {
    RopeTensor t[ROPE_MAX_TENSORS];
    unsigned long long freq[ROPE_MAX_PAIRS];           // turns per position, a 64-bit fraction
    unsigned char axis[ROPE_MAX_PAIRS];
    const int* pos;                                    // [pos_rows, ld_pos]; row r takes row r % pos_rows
    int n, heads, rows, pos_rows, ld_pos, dim, rot, block_rows, row_threads, inverse;
    float amplitude;
};

// What a thread takes of a head: eight elements of either side of the pairs (HALF), eight elements, or pieces of the part that does not turn.
struct RopeUnits {
    int per_head, turned, slots;                       // units of a head, those that turn, (cos, sin) places of a row
};
__host__ __device__ inline RopeUnits rope_units(bool half, int dim, int rot) {
    const int pairs = rot / 2, each = half ? 8 : 4, turned = (pairs + each - 1) / each;
    return {half ? turned + (dim - rot) / 8 : dim / 8, turned, turned * each};
}
enum { ROPE_ELEMENTS, ROPE_PIECES, ROPE_SHIFTED };       // see the two kernels
inline int rope_way(bool wide, bool half, int rot) { return !wide ? ROPE_ELEMENTS : half && rot % 16 ? ROPE_SHIFTED : ROPE_PIECES; }
// Heads whose loads a thread has under way together. Measured on B200, 16-bit, 2 and 4: 4096 x (16 + 16) heads of 128 half 12.5, 13.6 us, interleaved 14.1, 12.8; shifted, 126 of
// 128, 16 + 4 heads, 15.6, 14.7. fp32 half, 1 and 2: 1536 rows 10.6, 10.3; shifted 21.5, 22.6
__host__ __device__ constexpr int rope_together(int way, bool half, int elem) {
    return way == ROPE_SHIFTED ? (elem == 2 ? 4 : 1) : elem == 2 && !half ? 4 : 2;
}
// Rows of a thread block and the threads of each. Where a row is short, as many as fit. Else 1, or 2 or 4 where more of the loads that the threads could have under way are
// then real ones, and all SMs have eight blocks even so: with fewer, rows side by side instead of one behind the other are faster. Measured on B200, 1, 2 and 4 rows,
// the fullest one marked: 8190 rows, 16 + 4 heads of 128 interleaved bf16 19.4, 18.0, 16.3*; 4096 rows, 16 + 16 heads of 64 half bf16 9.0, 7.4*, 8.0; 8 + 8 of 128 interleaved fp16
// 10.7, 9.2*, 9.0, and 1024 such rows 4.4*, 5.8, 5.7; 16 + 16 of 128 12.8*, 13.1, 14.1.
inline void rope_split(int way, bool half, int elem, int dim, int rot, int heads, long long rows, int sm_count, int& block_rows, int& row_threads) {
    block_rows = 1;
    row_threads = ROPE_THREADS;
    if (way == ROPE_ELEMENTS) return;
    const int per_head = way == ROPE_SHIFTED ? dim / 8 : rope_units(half, dim, rot).per_head, all = per_head * heads, together = rope_together(way, half, elem);
    if (2 * all <= ROPE_THREADS) {
        row_threads = all;
        block_rows = ROPE_THREADS / all;
        return;
    }
    long long best_of = 0, best_turns = 1;                 // all / turns: the share of real loads
    for (int n = 1; n <= 4 && rows >= (n > 1 ? 8LL * n * sm_count : 0) && per_head * n <= ROPE_THREADS; n *= 2) {
        const int threads = ROPE_THREADS / n, at_once = threads / per_head * together;
        const long long turns = (long long)((heads + at_once - 1) / at_once) * together * threads;
        if (all * best_turns > best_of * turns) { best_of = all; best_turns = turns; block_rows = n; row_threads = threads; }
    }
}

// (cos, sin) of the rows of a thread block, a row's `stride` apart; a thread keeps its pair, so that it fetches one frequency. each > 1: the pairs of a unit of `each`
// lie `turned` apart, those of neighbouring units side by side, so that neighbouring lanes read neighbouring words
__device__ __forceinline__ void rope_sines(const RopeParams& p, float2* cs, unsigned row0, int rows, int stride, int each, int turned) {
    const int pairs = p.rot >> 1, per = ROPE_THREADS / pairs, f = threadIdx.x % pairs;
    int r = threadIdx.x / pairs;
    if (r >= per) return;
    const unsigned long long freq = p.freq[f];
    const int axis = p.axis[f];
    float2* const at = cs + (f % each) * turned + f / each;
    for (; r < rows; r += per) {
        const int pos = p.pos[(size_t)((row0 + (unsigned)r) % (unsigned)p.pos_rows) * p.ld_pos + axis];
        const unsigned long long turn = (unsigned long long)(long long)pos * freq;
        float sn, cn;
        sincospif((float)(int)(turn >> 32) * 0x1p-31f, &sn, &cn);     // in half turns, [-1, 1)
        at[r * stride] = make_float2(cn * p.amplitude, (p.inverse ? -sn : sn) * p.amplitude);
    }
}
// A pair turned, written out down to which product the sum is fused with, so that pieces and elements give the same bits whatever stands around them
__device__ __forceinline__ float rope_a(float a, float b, float2 z) { return fmaf(a, z.x, -__fmul_rn(b, z.y)); }
__device__ __forceinline__ float rope_b(float a, float b, float2 z) { return fmaf(a, z.y, __fmul_rn(b, z.x)); }
// where head v of a row lies
template <typename T>
__device__ __forceinline__ void rope_head(const RopeParams& p, unsigned row, int v, const T*& src, T*& dst) {
    const RopeTensor* t = &p.t[0];
#pragma unroll
    for (int k = 1; k < ROPE_MAX_TENSORS; k++)
        if (k < p.n && v >= p.t[k].first) t = &p.t[k];
    src = static_cast<const T*>(t->x) + (size_t)row * t->ld_x + (v - t->first) * p.dim;
    dst = static_cast<T*>(t->y) + (size_t)row * t->ld_y + (v - t->first) * p.dim;
}
// Which unit of which head of which of the block's rows a thread takes, and how many heads on its next one is (the same for the whole block); the units of a head are neighbouring threads'
struct RopePlace {
    int r, v, s, step;
    bool busy;
    __device__ __forceinline__ RopePlace(const RopeParams& p, int per_head, int rows) {
        r = threadIdx.x / p.row_threads;
        const int j = threadIdx.x - r * p.row_threads;
        v = j / per_head;
        s = j - v * per_head;
        step = p.row_threads / per_head;
        busy = r < rows && v < step && v < p.heads;
    }
};

// CUT: the part of the head that turns ends inside a piece (interleaved, rot no multiple of eight), whose other pairs are copied. Not asked in the kernel without
// it: 8190 rows of 16 + 4 heads, bf16, 96 of 128 15.1 us, with it 15.7.
// VEC (ROPE_PIECES): in pieces of eight elements, where every row starts on 16 bytes and a head (HALF: either side of the pairs too) is whole pieces; else
// (ROPE_ELEMENTS) a warp takes a head, element by element.
template <typename T, bool HALF, bool VEC, bool CUT = false>
__global__ void __launch_bounds__(ROPE_THREADS)
rope_kernel(const __grid_constant__ RopeParams p) {
    __shared__ float2 cs[ROPE_SLOTS];
    constexpr int EACH = HALF ? 8 : 4;
    pdl_launch();
    pdl_wait();
    const int pairs = p.rot >> 1;
    const RopeUnits un = rope_units(HALF, p.dim, p.rot);
    const int stride = VEC ? un.slots : pairs;
    const unsigned row0 = blockIdx.x * (unsigned)p.block_rows;
    const int rows = (int)min((unsigned)p.block_rows, (unsigned)p.rows - row0);
    if constexpr (VEC) {
        const RopePlace at(p, un.per_head, rows);
        const int r = at.r, s = at.s, step = at.step;
        int v = at.v;
        const unsigned row = row0 + (unsigned)r;
        const bool turns = s < un.turned;
        constexpr int U = rope_together(ROPE_PIECES, HALF, sizeof(T));
        const int ca = HALF && !turns ? p.rot + 8 * (s - un.turned) : 8 * s, cb = pairs + 8 * s;
        Raw8<T> a[U], b[U];
        T* dst[U];
        auto load = [&]() {
#pragma unroll
            for (int i = 0; i < U; i++) {
                if (v + i * step >= p.heads) break;
                const T* src;
                rope_head(p, row, v + i * step, src, dst[i]);
                a[i] = Io<T>::raw8(src + ca);
                if (HALF && turns) b[i] = Io<T>::raw8(src + cb);
            }
        };
        if (at.busy) load();                           // under the sines
        rope_sines(p, cs, row0, rows, stride, EACH, un.turned);
        __syncthreads();
        if (!at.busy) return;
        const int mine = CUT ? pairs - EACH * s : EACH;        // pairs of the unit that turn
        float2 z[EACH];
#pragma unroll
        for (int e = 0; e < EACH; e++) z[e] = turns && e < mine ? cs[r * stride + e * un.turned + s] : make_float2(1.f, 0.f);
        while (true) {
#pragma unroll
            for (int i = 0; i < U; i++) {
                if (v + i * step >= p.heads) break;
                if (!turns) { Io<T>::st8(dst[i] + ca, Io<T>::f8(a[i])); continue; }
                F8 x = Io<T>::f8(a[i]);
                if constexpr (HALF) {
                    F8 y = Io<T>::f8(b[i]);
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float t = x.v[e];
                        x.v[e] = rope_a(t, y.v[e], z[e]);
                        y.v[e] = rope_b(t, y.v[e], z[e]);
                    }
                    Io<T>::st8(dst[i] + cb, y);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float t = x.v[2 * e], u = x.v[2 * e + 1];
                        x.v[2 * e] = e < mine ? rope_a(t, u, z[e]) : t;
                        x.v[2 * e + 1] = e < mine ? rope_b(t, u, z[e]) : u;
                    }
                }
                Io<T>::st8(dst[i] + ca, x);
            }
            v += U * step;
            if (v >= p.heads) break;
            load();
        }
    } else {
        rope_sines(p, cs, row0, rows, stride, 1, 1);
        __syncthreads();
        const int lane = threadIdx.x & 31;
        for (int v = threadIdx.x >> 5; v < p.heads; v += ROPE_THREADS / 32) {
            const T* src;
            T* dst;
            rope_head(p, row0, v, src, dst);
            for (int s = lane; s < pairs; s += 32) {
                const int ia = HALF ? s : 2 * s, ib = HALF ? pairs + s : 2 * s + 1;
                const float2 z = cs[s];
                const float x = to_f32(src[ia]), y = to_f32(src[ib]);
                dst[ia] = from_f32<T>(rope_a(x, y, z));
                dst[ib] = from_f32<T>(rope_b(x, y, z));
            }
            for (int c = p.rot + lane; c < p.dim; c += 32) dst[c] = src[c];
        }
    }
}

// Halves of pairs where no piece of eight begins with the second one (rot / 2 no multiple of eight): a thread takes eight elements of a head, and their partners one by one
// out of shared memory, where the block's heads lie for the while. A block has read its heads before it writes one, so the output may be the input. Measured on
// B200, a warp per head, element by element -> this: 4096 rows, 126 of 128, 16 + 4 heads, fp16 23.3 -> 14.7 us, fp32 29.3 -> 21.5 (3.9 TB/s); 34 of 128, 16 + 16 heads, fp16
// 43.7 -> 17.2 (3.9). Partners as two pieces shifted by a run-time count: 37 us for the first. What bounds it is the instructions of a partner apiece.
template <typename T>
__global__ void __launch_bounds__(ROPE_THREADS, sizeof(T) == 2 ? 1 : 8)
rope_shifted_kernel(const __grid_constant__ RopeParams p) {
    constexpr int U = rope_together(ROPE_SHIFTED, true, sizeof(T));
    __shared__ float2 cs[ROPE_SLOTS];                  // a row has 8 turned <= dim of them, and block_rows * heads * dim / 8 <= ROPE_THREADS (or block_rows = 1, dim <= 256)
    __shared__ Raw8<T> stage[U * ROPE_THREADS];
    pdl_launch();
    pdl_wait();
    const int pairs = p.rot >> 1, per_head = p.dim >> 3, turned = (pairs + 7) >> 3;
    const unsigned row0 = blockIdx.x * (unsigned)p.block_rows;
    const int rows = (int)min((unsigned)p.block_rows, (unsigned)p.rows - row0);
    const RopePlace at(p, per_head, rows);
    const unsigned row = row0 + (unsigned)at.r;
    const int c0 = 8 * at.s;
    Raw8<T> a[U];
    T* dst[U];
    float2 z[8];
    for (int first = 0; first < p.heads; first += U * at.step) {          // `first` and `step` are the same for the whole block
        const int v = first + at.v;
#pragma unroll
        for (int i = 0; i < U; i++) {
            if (!at.busy || v + i * at.step >= p.heads) break;
            const T* src;
            rope_head(p, row, v + i * at.step, src, dst[i]);
            a[i] = Io<T>::raw8(src + c0);
        }
        if (first == 0) rope_sines(p, cs, row0, rows, 8 * turned, 8, turned);
        else __syncthreads();                                             // the heads before are done with
#pragma unroll
        for (int i = 0; i < U; i++) {
            if (!at.busy || v + i * at.step >= p.heads) break;
            stage[i * ROPE_THREADS + threadIdx.x] = a[i];
        }
        __syncthreads();
        if (!at.busy) continue;
        const int left = p.rot - c0, low = pairs - c0;                    // elements of the piece that turn, those of the first half
        if (first == 0) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int f = min(c0 + e - (e < low ? 0 : pairs), pairs - 1);
                z[e] = cs[at.r * 8 * turned + (f & 7) * turned + (f >> 3)];
                z[e].y = e < low ? -z[e].y : z[e].y;
            }
        }
#pragma unroll
        for (int i = 0; i < U; i++) {
            if (v + i * at.step >= p.heads) break;
            F8 x = Io<T>::f8(a[i]);
            if (left > 0) {
                const T* const own = reinterpret_cast<const T*>(stage + i * ROPE_THREADS + threadIdx.x);
                const T* const to = own + pairs;
                const T* const from = own - pairs;
#pragma unroll
                for (int e = 0; e < 8; e++) {                             // a partner lies in the head whatever e; it is taken where e turns
                    const float y = to_f32((e < low ? to : from)[e]), t = fmaf(x.v[e], z[e].x, __fmul_rn(y, z[e].y));
                    x.v[e] = e < left ? t : x.v[e];
                }
            }
            Io<T>::st8(dst[i] + c0, x);
        }
    }
}

}  // namespace kb
