// 4-bit floating point in blocks (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign) that share a scale: to and from it.
//   MX4  blocks of 32 columns, a = max |x|, s = 2^(floor(log2 a) - 2) (no less than 2^-127), stored as its exponent + 127 (E8M0)
//   NV4  blocks of 16 columns, y = x 2^-exp, s = max |y| / 6 rounded to E4M3 (no less than 2^-9, no more than 448); `exp` belongs to the whole matrix
// and each element is x / s (y / s) rounded to the nearest of the eight values, ties to the even code, beyond 6 to 6. Every one of these is
// decided exactly, so a value has one code whatever computes it: the quotients take one step of correction (Markstein, 1990:
// q0 = y r, q = q0 + r (y - q0 s) with a fused remainder), which makes a y that lies on a border (1.25 s, ...) give the border itself; a y
// next to one is at least a 24-bit step away from it, more than the rounding of q. A block that holds an infinity or a NaN gets a NaN for its scale.
//
// Layout of a matrix [rows, cols]: codes two to a byte, the even column in the low half, rows of `ld` bytes, filled with zeros up to
// a multiple of 32 columns. Scales in pieces of 512 bytes, 128 rows x 4 blocks, as the tensor cores' copy into TMEM reads them (32 lanes x 16
// bytes): row r, block b at byte ((r / 128) pieces + b / 4) 512 + (r % 32) 16 + (r / 32 % 4) 4 + b % 4; pieces = ceil(blocks / 4), the
// scales of blocks behind the last one are zeros, those of rows behind the last one are not touched.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "attn_sm100.cuh"   // ST_RANGE
#include "prep.cuh"   // Io
#include "ptx.cuh"

namespace kb {

constexpr int FMT_MX4 = 0, FMT_NV4 = 1;
__host__ __device__ constexpr int q4_block(int fmt) { return fmt == FMT_MX4 ? 32 : 16; }
__host__ __device__ constexpr int q4_pieces(int cols, int fmt) { return (cols + 4 * q4_block(fmt) - 1) / (4 * q4_block(fmt)); }   // of a row block
__host__ __device__ constexpr int q4_row_bytes(int cols) { return (cols + 31) / 32 * 16; }
__device__ __forceinline__ size_t q4_scale_at(int row, int piece, int pieces) {   // the four scales of a piece
    return ((size_t)(row >> 7) * pieces + piece) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// 2^e, e in [-126, 127]
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// four pairs of codes from eight numbers (already divided by their scale), element i in bits [4 i, 4 i + 4)
__device__ __forceinline__ uint32_t e2m1_pack8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// eight codes as four half2 (every value is one of fp16)
__device__ __forceinline__ void e2m1_unpack8(uint32_t codes, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(codes));
}
__device__ __forceinline__ uint32_t e4m3_byte(float v) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(v));
    return r & 0xffu;
}
__device__ __forceinline__ float e4m3_value(uint32_t byte) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)byte));
    return __half2float(__ushort_as_half((uint16_t)h));
}
// what a scale byte stands for; MX4's smallest, 2^-127, is a subnormal number
template <int FMT>
__device__ __forceinline__ float q4_scale_value(uint32_t byte) {
    if (FMT == FMT_NV4) return e4m3_value(byte);
    return byte == 0u ? __uint_as_float(0x00400000u) : byte == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(byte << 23);
}

// The scale of a block whose largest |x| has these bits: its byte, and with 2^exp what elements are divided by (s) and multiplied with (r ~ 1 / s).
template <int FMT>
struct BlockScale {
    uint32_t byte;
    float s, r;
    // down, up = 2^-exp, 2^exp of the matrix (NV4)
    __device__ __forceinline__ BlockScale(uint32_t abs_bits, float down, float up) {
        if (FMT == FMT_MX4) {
            const uint32_t e = abs_bits >> 23;
            byte = e > 2u ? e - 2u : 0u;                       // floor(log2 a) + 127 - 2
            r = __uint_as_float((254u - byte) << 23);
            s = 0.f;                                           // powers of two: a product is exact
        } else {
            const float a = __uint_as_float(abs_bits) * down, sixth = 1.f / 6.f;
            float q = a * sixth;
            q = fmaf(fmaf(-q, 6.f, a), sixth, q);
            byte = max(e4m3_byte(q), 1u);
            s = e4m3_value(byte) * up;
            r = __fdividef(1.f, s);                            // its last bit does not matter: the correction has the rest
        }
        if (abs_bits >= 0x7f800000u) byte = FMT == FMT_MX4 ? 255u : 127u;
    }
    // eight elements, as packed pairs, to eight codes
    __device__ __forceinline__ uint32_t codes(const uint64_t* v) const {
        const uint64_t r2 = pack2(r, r), ns2 = pack2(-s, -s);
        float q[8];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            uint64_t z = mul2(v[e], r2);
            if (FMT == FMT_NV4) z = fma2(fma2(z, ns2, v[e]), r2, z);
            unpack2(z, q[2 * e], q[2 * e + 1]);
        }
        return e2m1_pack8(q);
    }
};

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Rows that do not start on 16 bytes. One thread's eight elements one by one would touch a different 16 bytes in every lane, eight times over; so a
// warp (or `width` of its lanes) takes its width x 8 columns across, element j of a lane being column j * width + lane, and turns them round in shared memory.
// Measured on B200, one by one -> across: 4001 x 8190 bf16 to NV4 30.2 -> 24.2 us, back to fp16 54.6 -> 18.8, transposed 94 -> 31; 4001 x 4099 fp32 to NV4 20.7 -> 15.9;
// dropout (dropout.cuh) of 4000 x 8190 fp16 85.8 -> 42.7, 1000 x 2047 9.7 -> 4.2, 2000 x 4099 fp32 22.9 -> 17.0.
template <typename T>
__device__ __forceinline__ Raw8<T> load_across(const T* row, int first, int cols, int lane, int width) {      // zeros behind the last column
    Raw8<T> r;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int c = first + j * width + lane;
        reinterpret_cast<T*>(r.u)[j] = c < cols ? row[c] : from_f32<T>(0.f);
    }
    return r;
}
// `tile`: width places; the whole warp calls
template <typename T>
__device__ __forceinline__ Raw8<T> across_to_own(const Raw8<T>& r, Raw8<T>* tile, int lane, int width) {
#pragma unroll
    for (int j = 0; j < 8; j++) reinterpret_cast<T*>(tile)[j * width + lane] = reinterpret_cast<const T*>(r.u)[j];
    __syncwarp();
    return tile[lane];
}
template <typename T>
__device__ __forceinline__ void store_across(const Raw8<T>& own, Raw8<T>* tile, T* row, int first, int cols, int lane, int width) {
    tile[lane] = own;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int c = first + j * width + lane;
        if (c < cols) row[c] = reinterpret_cast<const T*>(tile)[j * width + lane];
    }
}

// eight elements from column c of a row that starts on 16 bytes, zeros behind the last column
template <typename T>
__device__ __forceinline__ Raw8<T> load8_raw(const T* row, int c, int cols) {
    if (c + 8 <= cols) return Io<T>::raw8(row + c);
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < 8; i++) reinterpret_cast<T*>(r.u)[i] = c + i < cols ? row[c + i] : from_f32<T>(0.f);
    return r;
}
template <typename T>
__device__ __forceinline__ void store8(T* row, int c, int cols, const F8& f) {
    if (c + 8 <= cols) { Io<T>::st8(row + c, f); return; }
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (c + i < cols) row[c + i] = from_f32<T>(f.v[i]);
}

struct Quant4Params {
    const void* x;               // [rows, ld_x]
    void* y;                     // dequant: [rows, ld_x], transposed [cols, ld_x]
    uint8_t* codes;
    uint8_t* scales;
    int rows, cols, ld_x, ld;    // ld: bytes of a row of codes
    int pieces;                  // of a row block
    int exp;
    bool wide;
    uint32_t* status;            // dequant transposed to fp16: set ST_RANGE where a value is not one of fp16's (null: not asked)
};

// A lane takes eight columns, so that a block is two (NV4) or four (MX4) lanes, which meet by shuffles; a warp 256 columns side by side, SEGS times, its loads
// first. Bound by memory: 16-bit rows 2 bytes read and 0.56 written per element. SEGS is 4 for 16-bit matrices of at least Q4_LARGE elements, where thread blocks of
// 2 come and go too fast, and else 2. Measured on B200, 2 -> 4, NV4 and MX4: 4096 x 8192 fp16 20.1 -> 18.3 us, 18.9 -> 15.7; 4096 x 2048 6.6 -> 6.7, 6.3 -> 6.0;
// 1536 x 2048 3.2 -> 4.2, 3.2 -> 3.7. 8192 x 2048 fp32 13.4 and 13.1 us (5.7 TB/s) either way.
constexpr int Q4_THREADS = 128;
constexpr long long Q4_LARGE = 12LL << 20;

// WIDE: every row of x starts on 16 bytes
template <typename T, int FMT, int SEGS, bool WIDE>
__global__ void __launch_bounds__(Q4_THREADS, SEGS == 2 ? 12 : 10)
quant4_kernel(const Quant4Params p) {
    pdl_launch();
    pdl_wait();
    const unsigned row = blockIdx.x * (Q4_THREADS / 32) + (threadIdx.x >> 5);
    if (row >= (unsigned)p.rows) return;
    const int lane = threadIdx.x & 31, c0 = (int)blockIdx.y * (SEGS * 256) + lane * 8;
    const T* const src = static_cast<const T*>(p.x) + (size_t)row * p.ld_x;
    const float down = pow2f(-p.exp), up = pow2f(p.exp);
    const uint32_t limit = __float_as_uint(8192.f * up);       // beyond 6 x 448 2^exp all is 6 times the largest scale; |x| 2^-exp itself might not be an fp32 number
    __shared__ Raw8<T> tiles[WIDE ? 1 : Q4_THREADS];
    Raw8<T> raw[SEGS];
#pragma unroll
    for (int i = 0; i < SEGS; i++) raw[i] = WIDE ? load8_raw(src, c0 + i * 256, p.cols) : load_across(src, c0 - lane * 8 + i * 256, p.cols, lane, 32);
#pragma unroll
    for (int i = 0; i < SEGS; i++) {
        const int c = c0 + i * 256;
        if (c - lane * 8 >= p.cols) break;                     // the whole warp is behind the last column (a piece never begins there)
        if (!WIDE) {
            if (i > 0) __syncwarp();
            raw[i] = across_to_own(raw[i], tiles + threadIdx.x - lane, lane, 32);
        }
        F8 f = Io<T>::f8(raw[i]);
        float big = max3_abs_nan(f.v[0], f.v[1], f.v[2]);
        big = max3_abs_nan(big, f.v[3], f.v[4]);
        big = max3_abs_nan(big, f.v[5], f.v[6]);
        uint32_t top = __float_as_uint(max3_abs_nan(big, f.v[7], 0.f)) & 0x7fffffffu;
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        if (FMT == FMT_MX4) top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (FMT == FMT_NV4 && !std::is_same<T, __half>::value && top > limit && top < 0x7f800000u) {      // (an fp16 number is below 2^16)
            top = limit;
#pragma unroll
            for (int e = 0; e < 8; e++) f.v[e] = fminf(fmaxf(f.v[e], -__uint_as_float(limit)), __uint_as_float(limit));
        }
        const BlockScale<FMT> bs(top, down, up);
        uint64_t v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = pack2(f.v[2 * e], f.v[2 * e + 1]);
        if (c < q4_row_bytes(p.cols) * 2) *reinterpret_cast<uint32_t*>(p.codes + (size_t)row * p.ld + (c >> 1)) = bs.codes(v);
        // the four scales of a piece, 8 (NV4) or 16 lanes, meet in its first lane
        constexpr int STEP = q4_block(FMT) / 8;
        uint32_t word = c < p.cols ? bs.byte << (8 * ((lane / STEP) & 3)) : 0u;
        word |= __shfl_xor_sync(0xffffffffu, word, STEP);
        word |= __shfl_xor_sync(0xffffffffu, word, 2 * STEP);
        const int piece = c / (4 * q4_block(FMT));
        if (lane % (4 * STEP) == 0 && piece < p.pieces) *reinterpret_cast<uint32_t*>(p.scales + q4_scale_at(row, piece, p.pieces)) = word;
    }
}

// eight codes from column c (a multiple of 8) of a row, and their scale's byte
struct Q4Raw { uint32_t codes, scale; };
template <int FMT>
__device__ __forceinline__ Q4Raw q4_load8(const Quant4Params& p, int row, int c) {
    const int b = c / q4_block(FMT);
    return {*reinterpret_cast<const uint32_t*>(p.codes + (size_t)row * p.ld + (c >> 1)), p.scales[q4_scale_at(row, b >> 2, p.pieces) + (b & 3)]};
}
// The values in T, as they lie in memory; up = 2^exp. In fp16 the product is taken in fp16 where the scale is one of its numbers: the same single rounding.
template <typename T, int FMT>
__device__ __forceinline__ Raw8<T> q4_values8(const Q4Raw& q, float up) {
    uint32_t h[4];
    e2m1_unpack8(q.codes, h);
    const float s = q4_scale_value<FMT>(q.scale) * up;
    Raw8<T> out;
    if constexpr (std::is_same<T, __half>::value) {
        const __half sh = __float2half_rn(s);
        if (__half2float(sh) == s) {
            const __half2 s2 = __half2half2(sh);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&h[i]), s2);
                h[i] = *reinterpret_cast<const uint32_t*>(&v);
            }
            out.u[0] = make_uint4(h[0], h[1], h[2], h[3]);
            return out;
        }
    }
    F8 f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        f.v[2 * i] = v.x * s;
        f.v[2 * i + 1] = v.y * s;
    }
    Io<T>::st8(reinterpret_cast<T*>(out.u), f);
    return out;
}
// A lane takes 16 bytes of output (fp32: half of eight codes), so that every store of a warp is 512 bytes in a row, or where rows do not start on 16 bytes as many stores
// of an element apiece as a lane has. Measured on B200, fp16, 512 columns of a warp -> 1024: 4096 x 8192 18.5 -> 15.8 us, 8192 x 2048 10.0 -> 8.6, 1536 x 2048 3.0 -> 3.0; fp32 the
// other way: 1536 x 2048 4.6 -> 5.0, 8192 x 2048 14.2 -> 14.8.
template <typename T> __host__ __device__ constexpr int deq_cols() { return sizeof(T) == 2 ? 1024 : 512; }   // columns of a warp
template <typename T, int FMT>
__global__ void __launch_bounds__(Q4_THREADS)
dequant4_kernel(const Quant4Params p) {
    constexpr int EACH = 16 / sizeof(T), COLS = deq_cols<T>(), N = COLS / (32 * EACH);
    pdl_launch();
    pdl_wait();
    const unsigned row = blockIdx.x * (Q4_THREADS / 32) + (threadIdx.x >> 5);
    if (row >= (unsigned)p.rows) return;
    const int first = (int)blockIdx.y * COLS, lane = threadIdx.x & 31;
    T* const dst = static_cast<T*>(p.y) + (size_t)row * p.ld_x;
    const float up = pow2f(p.exp);
    __shared__ uint4 tiles[Q4_THREADS];                       // of rows that do not start on 16 bytes
    Q4Raw q[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int c = first + (i * 32 + lane) * EACH;
        q[i] = c < p.cols ? q4_load8<FMT>(p, (int)row, c & ~7) : Q4Raw{0u, 0u};
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int c = first + (i * 32 + lane) * EACH;
        if (c - lane * EACH >= p.cols) break;
        const Raw8<T> v = q4_values8<T, FMT>(q[i], up);
        const uint4 out = EACH == 8 ? v.u[0] : (c & 4) ? v.u[sizeof(T) / 2 - 1] : v.u[0];
        if (!p.wide) {
            uint4* const tile = tiles + (threadIdx.x - lane);
            if (i > 0) __syncwarp();
            tile[lane] = out;
            __syncwarp();
#pragma unroll
            for (int j = 0; j < EACH; j++) {
                const int col = c - lane * EACH + j * 32 + lane;
                if (col < p.cols) dst[col] = reinterpret_cast<const T*>(tile)[j * 32 + lane];
            }
        } else if (c + EACH <= p.cols) *reinterpret_cast<uint4*>(dst + c) = out;
        else
#pragma unroll
            for (int e = 0; e < EACH; e++)
                if (c + e < p.cols) dst[c + e] = reinterpret_cast<const T*>(&out)[e];
    }
}

// The transpose [cols, ld_x], through shared memory in tiles of 128 rows x 64 columns: a thread decodes sixteen columns (one scale) of two rows side by side, which
// become sixteen pairs along rows of the transpose. What the gradient of a projection's input multiplies with. 8192 x 2048 to fp16 11.3 us (3.8 TB/s), 4096 x 8192 19.4;
// in tiles of 64 x 64 with eight columns per thread 14.0 and 25.8.
constexpr int Q4_TILE_R = 128, Q4_TILE_C = 64, Q4_TILE_LD = Q4_TILE_R + 8;      // a tile row in shared memory starts on 16 bytes, four banks further
template <typename T, int FMT>
__global__ void __launch_bounds__(256)
dequant4_t_kernel(const Quant4Params p) {
    __shared__ __align__(16) T tile[Q4_TILE_C * Q4_TILE_LD];
    pdl_launch();
    pdl_wait();
    const int tiles_c = (p.cols + Q4_TILE_C - 1) / Q4_TILE_C;
    const int r0 = (int)(blockIdx.x / (unsigned)tiles_c) * Q4_TILE_R, k0 = (int)(blockIdx.x % (unsigned)tiles_c) * Q4_TILE_C;
    const int pair = threadIdx.x & 63, kg = threadIdx.x >> 6, c = k0 + 16 * kg;
    const float up = pow2f(p.exp);
    uint2 codes[2];
    uint32_t scale[2];
    bool rounded = false;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int r = r0 + 2 * pair + i, b = c / q4_block(FMT);
        const bool in = r < p.rows && c < p.cols;
        codes[i] = in ? *reinterpret_cast<const uint2*>(p.codes + (size_t)r * p.ld + (c >> 1)) : make_uint2(0u, 0u);
        scale[i] = in ? p.scales[q4_scale_at(r, b >> 2, p.pieces) + (b & 3)] : 0u;
        // a half of the scale down to 2^-24, six of it up to 49152; a NaN is one of fp16 as well, and zeros are whatever their scale
        rounded |= FMT == FMT_MX4 && (scale[i] < 127u - 23u || scale[i] > 127u + 13u) && scale[i] != 255u && ((codes[i].x | codes[i].y) & 0x77777777u) != 0u;
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const Raw8<T> v0 = q4_values8<T, FMT>({h ? codes[0].y : codes[0].x, scale[0]}, up), v1 = q4_values8<T, FMT>({h ? codes[1].y : codes[1].x, scale[1]}, up);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            struct alignas(2 * sizeof(T)) Two { T a, b; } two = {reinterpret_cast<const T*>(v0.u)[e], reinterpret_cast<const T*>(v1.u)[e]};
            *reinterpret_cast<Two*>(&tile[(16 * kg + 8 * h + e) * Q4_TILE_LD + 2 * pair]) = two;
        }
    }
    if (std::is_same<T, __half>::value && FMT == FMT_MX4 && p.status) {
        if (__syncthreads_or(rounded) && threadIdx.x == 0) atomicOr(p.status, ST_RANGE);
    } else __syncthreads();
    if (!p.wide) {
        for (int i = threadIdx.x; i < Q4_TILE_C * Q4_TILE_R; i += 256) {
            const int k = i / Q4_TILE_R, n = i % Q4_TILE_R;
            if (k0 + k < p.cols && r0 + n < p.rows) static_cast<T*>(p.y)[(size_t)(k0 + k) * p.ld_x + r0 + n] = tile[k * Q4_TILE_LD + n];
        }
        return;
    }
    constexpr int EACH = 16 / sizeof(T), ACROSS = Q4_TILE_R / EACH;    // elements of 16 bytes
#pragma unroll
    for (int i = threadIdx.x; i < Q4_TILE_C * ACROSS; i += 256) {
        const int k = i / ACROSS, n = (i % ACROSS) * EACH, left = p.rows - r0 - n;
        if (k0 + k >= p.cols || left <= 0) continue;
        T* const dst = static_cast<T*>(p.y) + (size_t)(k0 + k) * p.ld_x + r0 + n;
        const uint4 v = *reinterpret_cast<const uint4*>(&tile[k * Q4_TILE_LD + n]);
        if (left >= EACH) *reinterpret_cast<uint4*>(dst) = v;
        else
#pragma unroll
            for (int e = 0; e < EACH; e++)
                if (e < left) dst[e] = reinterpret_cast<const T*>(&v)[e];
    }
}

}  // namespace kb
