// Rotary positions of up to four tensors (q and k, or their gradients) in one launch: of every head's first `rot` elements pair i turns by the
// angle t = pos[axis_i] f_i, (a, b) -> (a cos t - b sin t, b cos t + a sin t) * amplitude; the pairs are (i, i + rot / 2) (half) or
// (2 i, 2 i + 1) (interleaved), the rest of the head is copied. The inverse turns by -t: it is the gradient.
//
// The angle of a far position turns thousands of times, and fp32 has lost its fraction by then. Here a frequency is a 64-bit fraction of a turn
// and a position an integer, so their product modulo 2^64 IS the fraction of the turn, exactly, in two integer multiplications: the
// only rounding is that of the fraction to 32 bits (2^-32 of a turn) and the sine's own.
//
// Bound by memory. The sines of a row serve all of its heads: a thread block takes rows, its threads first fill shared memory with one
// (cos, sin) per row and pair, then turn the heads, eight elements of either side of the pairs at a time.
#pragma once
#include "quant4.cuh"   // load8, store8

namespace kb {

constexpr int ROPE_MAX_PAIRS = 128, ROPE_MAX_TENSORS = 4, ROPE_THREADS = 128;
constexpr int ROPE_SLOTS = 512;                        // (row, pair) places in shared memory

struct RopeTensor {
    const void* x;
    void* y;
    int heads, ld_x, ld_y;
};
struct RopeParams {
    RopeTensor t[ROPE_MAX_TENSORS];
    unsigned long long freq[ROPE_MAX_PAIRS];           // turns per position, a 64-bit fraction
    unsigned char axis[ROPE_MAX_PAIRS];
    const int* pos;                                    // [pos_rows, ld_pos]; row r takes row r % pos_rows
    int n, rows, pos_rows, ld_pos, dim, rot, block_rows, inverse;
    float amplitude;
    bool wide;                                         // rows of all tensors start on 16 bytes
};

// VEC: pieces of eight elements. HALF needs rot / 2 to be a multiple of 8 for it (the launch decides); else element by element.
template <typename T, bool HALF, bool VEC>
__global__ void __launch_bounds__(ROPE_THREADS)
rope_kernel(const __grid_constant__ RopeParams p) {
    __shared__ float2 cs[ROPE_SLOTS];
    pdl_launch();
    pdl_wait();
    const int pairs = p.rot >> 1;
    const long long row0 = (long long)blockIdx.x * p.block_rows;
    const int rows = (int)min((long long)p.block_rows, (long long)p.rows - row0);
    for (int i = threadIdx.x; i < rows * pairs; i += ROPE_THREADS) {
        const int r = i / pairs, f = i - r * pairs;
        const int pos = p.pos[(size_t)((row0 + r) % p.pos_rows) * p.ld_pos + p.axis[f]];
        const unsigned long long turn = (unsigned long long)(long long)pos * p.freq[f];
        float sn, cn;
        sincospif((float)(int)(turn >> 32) * 0x1p-31f, &sn, &cn);     // in half turns, [-1, 1)
        cs[i] = make_float2(cn * p.amplitude, (p.inverse ? -sn : sn) * p.amplitude);
    }
    __syncthreads();
    for (int k = 0; k < p.n; k++) {
        const RopeTensor& t = p.t[k];
        if (VEC) {
            const int pieces = p.dim >> 3, half = pairs >> 3, turned = HALF ? half : 0, rest = HALF ? pieces - 2 * half : pieces;
            const int per_head = turned + rest, n = rows * t.heads * per_head;     // HALF: `turned` pairs of pieces, then copied pieces
            for (int i = threadIdx.x; i < n; i += ROPE_THREADS) {
                const int r = i / (t.heads * per_head), j = i - r * (t.heads * per_head), h = j / per_head, s = j - h * per_head;
                const T* const src = static_cast<const T*>(t.x) + (size_t)(row0 + r) * t.ld_x + h * p.dim;
                T* const dst = static_cast<T*>(t.y) + (size_t)(row0 + r) * t.ld_y + h * p.dim;
                const float2* const row_cs = cs + r * pairs;
                if (HALF) {
                    if (s < turned) {
                        const F8 a = Io<T>::ld8(src + 8 * s), b = Io<T>::ld8(src + pairs + 8 * s);
                        F8 u, v;
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const float2 z = row_cs[8 * s + e];
                            u.v[e] = a.v[e] * z.x - b.v[e] * z.y;
                            v.v[e] = b.v[e] * z.x + a.v[e] * z.y;
                        }
                        Io<T>::st8(dst + 8 * s, u);
                        Io<T>::st8(dst + pairs + 8 * s, v);
                    } else {
                        const int c = p.rot + 8 * (s - turned);
                        Io<T>::st8(dst + c, Io<T>::ld8(src + c));
                    }
                } else {
                    F8 a = Io<T>::ld8(src + 8 * s);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if (4 * s + e >= pairs) continue;
                        const float2 z = row_cs[4 * s + e];
                        const float x = a.v[2 * e], y = a.v[2 * e + 1];
                        a.v[2 * e] = x * z.x - y * z.y;
                        a.v[2 * e + 1] = y * z.x + x * z.y;
                    }
                    Io<T>::st8(dst + 8 * s, a);
                }
            }
        } else {
            const int per_head = pairs + p.dim - p.rot, n = rows * t.heads * per_head;
            for (int i = threadIdx.x; i < n; i += ROPE_THREADS) {
                const int r = i / (t.heads * per_head), j = i - r * (t.heads * per_head), h = j / per_head, s = j - h * per_head;
                const T* const src = static_cast<const T*>(t.x) + (size_t)(row0 + r) * t.ld_x + h * p.dim;
                T* const dst = static_cast<T*>(t.y) + (size_t)(row0 + r) * t.ld_y + h * p.dim;
                if (s < pairs) {
                    const int ia = HALF ? s : 2 * s, ib = HALF ? pairs + s : 2 * s + 1;
                    const float2 z = cs[r * pairs + s];
                    const float x = to_f32(src[ia]), y = to_f32(src[ib]);
                    dst[ia] = from_f32<T>(x * z.x - y * z.y);
                    dst[ib] = from_f32<T>(y * z.x + x * z.y);
                } else {
                    const int c = p.rot + s - pairs;
                    dst[c] = src[c];
                }
            }
        }
    }
}

}  // namespace kb
