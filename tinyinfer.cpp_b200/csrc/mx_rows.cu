// Rows into the microscaled format (mx.cuh), out of it, and the root-mean-square norm whose output is in it.
//
// All three are bound by the bytes they move and, for few rows, by one round trip to memory; the first two come close to the
// limit of instructions too, so a thread's place costs no division (a block is a power of two of threads along a row) and
// conversions are the hardware's, two elements each.  A thread owns eight neighbouring elements at a time (16 bytes of
// bfloat16, 32 of float32), so a block of 32 is four lanes and a chunk of 128 sixteen: the block's largest magnitude is two
// shuffles, a chunk's four scale bytes meet in one lane, which stores them as a word.  Rows whose start or stride does not
// allow such accesses take a second form in which a warp walks a chunk with one element of each of its blocks a lane: every
// access is still 32 neighbours, the maximum is one redux.
#include <cuda_fp16.h>

#include "mx.cuh"

namespace {

using namespace mx;

constexpr int UNIT = 8;                 // elements of a thread

template <typename T> __device__ __forceinline__ void load_unit(const T* p, float (&v)[UNIT]);
template <> __device__ __forceinline__ void load_unit<bf16>(const bf16* p, float (&v)[UNIT]) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
template <> __device__ __forceinline__ void load_unit<float>(const float* p, float (&v)[UNIT]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void store_unit(float* p, const float (&v)[UNIT]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store_unit(bf16* p, const float (&v)[UNIT]) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 x = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const unsigned*>(&x);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Eight elements of a row from column c on; zeros from column k on.  `whole`: rows start on 16 bytes.
template <typename T> __device__ __forceinline__ void load_guarded(const T* row, int c, int k, bool whole, float (&v)[UNIT]) {
    if (whole && c + UNIT <= k) {
        load_unit(row + c, v);
    } else {
#pragma unroll
        for (int i = 0; i < UNIT; ++i) v[i] = c + i < k ? to_f32(row[c + i]) : 0.0f;
    }
}
template <typename T> __device__ __forceinline__ void store_guarded(T* row, int c, int k, bool whole, const float (&v)[UNIT]) {
    if (whole && c + UNIT <= k) {
        store_unit(row + c, v);
    } else {
#pragma unroll
        for (int i = 0; i < UNIT; ++i)
            if (c + i < k) row[c + i] = from_f32<T>(v[i]);
    }
}

// The largest magnitude's float32 bits.  Bits, not numbers: a NaN is larger than everything then.
__device__ __forceinline__ unsigned top_of(const float (&v)[UNIT]) {
    unsigned b[UNIT];
#pragma unroll
    for (int i = 0; i < UNIT; ++i) b[i] = __float_as_uint(v[i]) & 0x7fffffffu;
    const unsigned x = __vimax3_u32(b[0], b[1], b[2]), y = __vimax3_u32(b[3], b[4], b[5]);
    return max(__vimax3_u32(x, y, b[6]), b[7]);
}

// Codes and scales of a thread's eight elements at column c of a row; whole groups of sixteen neighbouring lanes call it
// together, c a multiple of 128 in the group's first lane.  `at`, `scale_word`: where the row's codes and the scale words of
// its chunks begin (a row's words are 512 bytes apart).
template <int BITS>
__device__ __forceinline__ void store_codes(const float (&v)[UNIT], int c, unsigned char* at, unsigned char* scale_words) {
    const unsigned half = 0xffffu << (threadIdx.x & 16);
    unsigned top = top_of(v);
    top = max(top, __shfl_xor_sync(half, top, 1));
    top = max(top, __shfl_xor_sync(half, top, 2));
    const unsigned s = scale_byte<BITS>(top);
    const float inv = scale_inverse(s);
    if (BITS == 8) {
        unsigned w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = codes_e4m3x2(v[4 * i] * inv, v[4 * i + 1] * inv) | codes_e4m3x2(v[4 * i + 2] * inv, v[4 * i + 3] * inv) << 16;
        *reinterpret_cast<uint2*>(at + c) = make_uint2(w[0], w[1]);
    } else {
        unsigned w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= codes_e2m1x2(v[2 * i] * inv, v[2 * i + 1] * inv) << (8 * i);
        *reinterpret_cast<unsigned*>(at + c / 2) = w;
    }
    unsigned word = s << (8 * (threadIdx.x >> 2 & 3));       // the four blocks of a chunk: lanes 0, 4, 8, 12 of sixteen
    word |= __shfl_xor_sync(half, word, 4);
    word |= __shfl_xor_sync(half, word, 8);
    if ((threadIdx.x & 15) == 0) *reinterpret_cast<unsigned*>(scale_words + (size_t)(c / CHUNK) * TILE_BYTES) = word;
}

// ---- quantisation --------------------------------------------------------------------------------

constexpr int QUANT_THREADS = 256;
constexpr int AHEAD = 2;                // units of a thread, all asked for before the first is used

// Where a thread of a row kernel works: 1 << shift threads lie along a row, QUANT_THREADS >> shift rows are in a block, and
// blockIdx.y counts segments of AHEAD << shift units of a row.
struct Place {
    long long row;
    int unit;                           // the first; the others follow at distances of 1 << shift
    __device__ explicit Place(int shift)
        : row(((long long)blockIdx.x << (8 - shift)) + (threadIdx.x >> shift)),
          unit((int)((blockIdx.y * AHEAD) << shift) + ((int)threadIdx.x & ((1 << shift) - 1))) {}
};

template <typename T, int BITS>
__global__ void __launch_bounds__(QUANT_THREADS)
mx_quantize_kernel(const T* x, long long ld, int rows, int k, int kp, unsigned char* codes, unsigned char* scales, int shift) {
    const Place me(shift);
    pdl_wait();
    if (me.row >= rows) return;                              // whole groups of sixteen lanes, here and below
    const T* from = x + (size_t)me.row * ld;
    float v[AHEAD][UNIT];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
        const int c = (me.unit + (u << shift)) * UNIT;
        if (c < kp) load_guarded(from, c, k, true, v[u]);
    }
    unsigned char *at = codes + (size_t)me.row * kp / (8 / BITS), *words = scales + scale_at((int)me.row, 0, kp / CHUNK);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
        const int c = (me.unit + (u << shift)) * UNIT;
        if (c < kp) store_codes<BITS>(v[u], c, at, words);
    }
}

// any start and stride: a warp takes a chunk, one element of each of its four blocks a lane
template <typename T, int BITS>
__global__ void __launch_bounds__(QUANT_THREADS)
mx_quantize_any_kernel(const T* x, long long ld, int rows, int k, int kp, unsigned char* codes, unsigned char* scales, int) {
    const unsigned chunks = (unsigned)kp / CHUNK, at = (blockIdx.x * QUANT_THREADS + threadIdx.x) / 32;
    const int lane = threadIdx.x & 31;
    pdl_wait();
    if (at >= (unsigned)rows * chunks) return;
    const int row = (int)(at / chunks), c = (int)(at % chunks) * CHUNK;
    const T* from = x + (size_t)row * ld;
    float v[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) v[b] = c + b * BLOCK + lane < k ? to_f32(from[c + b * BLOCK + lane]) : 0.0f;
    unsigned word = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const unsigned s = scale_byte<BITS>(__reduce_max_sync(0xffffffffu, __float_as_uint(v[b]) & 0x7fffffffu));
        word |= s << (8 * b);
        const float y = v[b] * scale_inverse(s);
        const size_t el = (size_t)row * kp + c + b * BLOCK + lane;
        if (BITS == 8) {
            codes[el] = (unsigned char)codes_e4m3x2(y, 0.0f);
        } else {
            const float next = __shfl_down_sync(0xffffffffu, y, 1);
            if (!(lane & 1)) codes[el / 2] = (unsigned char)codes_e2m1x2(y, next);
        }
    }
    if (lane == 0) *reinterpret_cast<unsigned*>(scales + scale_at(row, c / BLOCK, kp / CHUNK)) = word;
}

// ---- and back ------------------------------------------------------------------------------------

// eight codes as numbers without their scale; both element types are exact in float16
template <int BITS> __device__ __forceinline__ void values_of(uint2 w, float (&v)[UNIT]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        unsigned pair;
        if (BITS == 8)
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(pair) : "h"((unsigned short)((i < 2 ? w.x : w.y) >> (16 * (i & 1)))));
        else
            asm("{\n\t.reg .b8 b;\n\tcvt.u8.u32 b, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(pair) : "r"(w.x >> (8 * i)));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

template <typename T, int BITS>
__global__ void __launch_bounds__(QUANT_THREADS)
mx_dequantize_kernel(const unsigned char* codes, const unsigned char* scales, int rows, int k, int kp, T* out, long long ld,
                     int shift) {
    const Place me(shift);
    pdl_launch();
    pdl_wait();
    if (me.row >= rows) return;
    const unsigned char *at = codes + (size_t)me.row * kp / (8 / BITS), *words = scales + scale_at((int)me.row, 0, kp / CHUNK);
    uint2 w[AHEAD];
    unsigned s[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
        const int c = (me.unit + (u << shift)) * UNIT;
        if (c < k) {
            w[u] = BITS == 8 ? *reinterpret_cast<const uint2*>(at + c) : make_uint2(*reinterpret_cast<const unsigned*>(at + c / 2), 0);
            s[u] = words[(size_t)(c / CHUNK) * TILE_BYTES + c / BLOCK % 4];
        }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
        const int c = (me.unit + (u << shift)) * UNIT;
        if (c >= k) break;
        const float f = scale_value(s[u]);
        float v[UNIT];
        values_of<BITS>(w[u], v);
#pragma unroll
        for (int i = 0; i < UNIT; ++i) v[i] *= f;
        store_guarded(out + (size_t)me.row * ld, c, k, true, v);
    }
}

// rows of the output off 16 bytes
template <typename T, int BITS>
__global__ void __launch_bounds__(QUANT_THREADS)
mx_dequantize_any_kernel(const unsigned char* codes, const unsigned char* scales, int rows, int k, int kp, T* out, long long ld,
                         int) {
    const unsigned chunks = (unsigned)kp / CHUNK, at = (blockIdx.x * QUANT_THREADS + threadIdx.x) / 32;
    const int lane = threadIdx.x & 31;
    pdl_launch();
    pdl_wait();
    if (at >= (unsigned)rows * chunks) return;
    const int row = (int)(at / chunks), c = (int)(at % chunks) * CHUNK;
    const unsigned word = *reinterpret_cast<const unsigned*>(scales + scale_at(row, c / BLOCK, kp / CHUNK));
    const unsigned char* from = codes + ((size_t)row * kp + c) / (8 / BITS);
    T* to = out + (size_t)row * ld + c;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const int e = b * BLOCK + lane;
        const unsigned code = BITS == 8 ? from[e] : from[e / 2] >> (4 * (lane & 1)) & 15u;
        const float v = (BITS == 8 ? value_e4m3(code) : value_e2m1(code)) * scale_value(word >> (8 * b) & 255u);
        if (c + e < k) to[e] = from_f32<T>(v);
    }
}

// ---- the norm ------------------------------------------------------------------------------------

// One block a row, the row in registers: x += delta, sum of squares, then the codes.  UNITS units of eight elements a thread.
template <typename D, int BITS, int UNITS>
__global__ void __launch_bounds__(1024)
mx_rmsnorm_kernel(float* x, long long ldx, const D* delta, long long ldd, const float* __restrict__ weight, int k, int kp,
                  float eps, unsigned char* codes, unsigned char* scales, bool whole_x, bool whole_d, bool whole_w) {
    __shared__ float scratch[32];
    const int row = blockIdx.x;
    float* xr = x + (size_t)row * ldx;
    float v[UNITS][UNIT];
    pdl_launch();
    pdl_wait();
#pragma unroll
    for (int u = 0; u < UNITS; ++u) load_guarded(xr, (u * (int)blockDim.x + (int)threadIdx.x) * UNIT, k, whole_x, v[u]);
    if (delta != nullptr) {
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const int c = (u * (int)blockDim.x + (int)threadIdx.x) * UNIT;
            float d[UNIT];
            load_guarded(delta + (size_t)row * ldd, c, k, whole_d, d);
#pragma unroll
            for (int i = 0; i < UNIT; ++i) v[u][i] += d[i];
            store_guarded(xr, c, k, whole_x, v[u]);
        }
    }
    float sum = 0.0f;
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
#pragma unroll
        for (int i = 0; i < UNIT; ++i) sum = fmaf(v[u][i], v[u][i], sum);
    const float inv = rsqrtf(block_sum(sum, scratch) / (float)k + eps);
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const int c = (u * (int)blockDim.x + (int)threadIdx.x) * UNIT;
        if (c >= kp) break;                                  // whole groups of sixteen lanes: kp is a multiple of 128
        float w[UNIT];
        load_guarded(weight, c, k, whole_w, w);
#pragma unroll
        for (int i = 0; i < UNIT; ++i) v[u][i] = v[u][i] * inv * w[i];
        store_codes<BITS>(v[u], c, codes + (size_t)row * kp / (8 / BITS), scales + scale_at(row, 0, kp / CHUNK));
    }
}

bool whole_rows(const void* p, long long ld, int bytes) { return (uintptr_t)p % 16 == 0 && ld * bytes % 16 == 0; }

// The launch of a row kernel over `units` of eight elements a row: as many threads along a row as its units want at AHEAD
// each (16 to 256), or for rows off 16 bytes a warp a chunk.  False: too many for a grid.
struct Shape {
    dim3 grid;
    int shift = 8;
    bool set(bool whole, long long rows, int units, int chunks) {
        if (!whole) {
            const long long warps = rows * chunks;
            grid = dim3((unsigned)((warps + QUANT_THREADS / 32 - 1) / (QUANT_THREADS / 32)));
            return warps < (1LL << 27);
        }
        while (shift > 4 && AHEAD << (shift - 1) >= units) --shift;
        const long long in_block = QUANT_THREADS >> shift, segments = (units + (AHEAD << shift) - 1) / (AHEAD << shift);
        grid = dim3((unsigned)((rows + in_block - 1) / in_block), (unsigned)segments);
        return segments < 65536;
    }
};

template <typename T, int BITS>
int quantize(const void* x, long long ld, int rows, int k, int kp, void* codes, void* scales, void* stream) {
    const bool whole = whole_rows(x, ld, sizeof(T));
    Shape shape;
    TI_REQUIRE(shape.set(whole, rows, kp / UNIT, kp / CHUNK), "mx_quantize: %d rows of %d elements are too many", rows, k);
    ti_launch_pdl(whole ? mx_quantize_kernel<T, BITS> : mx_quantize_any_kernel<T, BITS>, shape.grid, QUANT_THREADS, 0,
                  (cudaStream_t)stream, (const T*)x, ld, rows, k, kp, (unsigned char*)codes, (unsigned char*)scales, shape.shift);
    return ti_check_launch("mx_quantize");
}

template <typename T, int BITS>
int dequantize(const void* codes, const void* scales, int rows, int k, int kp, void* out, long long ld, void* stream) {
    const bool whole = whole_rows(out, ld, sizeof(T));
    Shape shape;
    TI_REQUIRE(shape.set(whole, rows, (k + UNIT - 1) / UNIT, kp / CHUNK), "mx_dequantize: %d rows of %d elements are too many",
               rows, k);
    ti_launch_pdl(whole ? mx_dequantize_kernel<T, BITS> : mx_dequantize_any_kernel<T, BITS>, shape.grid, QUANT_THREADS, 0,
                  (cudaStream_t)stream, (const unsigned char*)codes, (const unsigned char*)scales, rows, k, kp, (T*)out, ld,
                  shape.shift);
    return ti_check_launch("mx_dequantize");
}

template <typename D, int BITS>
int rmsnorm(void* x, long long ldx, const void* delta, long long ldd, const void* weight, int rows, int k, int kp, float eps,
            void* codes, void* scales, void* stream) {
    const int units = kp / UNIT;
    const int per = units <= 256 ? 1 : units <= 512 ? 2 : 4;  // 256 threads a row, more units a thread, then more threads
    const int threads = ((units + per - 1) / per + 31) / 32 * 32;
    TI_REQUIRE(threads <= 1024, "mx_rmsnorm: rows of %d elements are longer than 32,768", k);
    auto kernel = per == 1 ? mx_rmsnorm_kernel<D, BITS, 1> : per == 2 ? mx_rmsnorm_kernel<D, BITS, 2> : mx_rmsnorm_kernel<D, BITS, 4>;
    ti_launch_pdl(kernel, (unsigned)rows, (unsigned)threads, 0, (cudaStream_t)stream, (float*)x, ldx, (const D*)delta, ldd,
                  (const float*)weight, k, kp, eps, (unsigned char*)codes, (unsigned char*)scales, whole_rows(x, ldx, 4),
                  whole_rows(delta, ldd, sizeof(D)), whole_rows(weight, 0, 4));
    return ti_check_launch("mx_rmsnorm");
}

int check_format(const char* who, int rows, int k, int kp, int bits, const void* codes, const void* scales) {
    TI_REQUIRE(rows >= 0 && k >= 1 && kp >= k && kp % CHUNK == 0, "%s: %d rows of %d elements padded to %d", who, rows, k, kp);
    TI_REQUIRE(bits == 4 || bits == 8, "%s: %d bits (4 and 8 are known)", who, bits);
    TI_REQUIRE((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0, "%s: codes and scales must start on 16 bytes", who);
    return 0;
}

}  // namespace

// codes, scales = x[rows, k] (x_code: TI_F32 or TI_BF16, ld elements between rows) in the format of `bits`
extern "C" int ti_mx_quantize(const void* x, int x_code, long long ld, int rows, int k, int kp, int bits, void* codes,
                              void* scales, void* stream) {
    if (int rc = check_format("mx_quantize", rows, k, kp, bits, codes, scales)) return rc;
    TI_REQUIRE(x_code == TI_F32 || x_code == TI_BF16, "mx_quantize: dtype code %d", x_code);
    if (rows == 0) return 0;
    auto run = x_code == TI_BF16 ? (bits == 8 ? quantize<bf16, 8> : quantize<bf16, 4>)
                                 : (bits == 8 ? quantize<float, 8> : quantize<float, 4>);
    return run(x, ld, rows, k, kp, codes, scales, stream);
}

// out[rows, k] = the numbers that codes and scales stand for
extern "C" int ti_mx_dequantize(const void* codes, const void* scales, int rows, int k, int kp, int bits, void* out,
                                int out_code, long long ld, void* stream) {
    if (int rc = check_format("mx_dequantize", rows, k, kp, bits, codes, scales)) return rc;
    TI_REQUIRE(out_code == TI_F32 || out_code == TI_BF16, "mx_dequantize: dtype code %d", out_code);
    if (rows == 0) return 0;
    auto run = out_code == TI_BF16 ? (bits == 8 ? dequantize<bf16, 8> : dequantize<bf16, 4>)
                                   : (bits == 8 ? dequantize<float, 8> : dequantize<float, 4>);
    return run(codes, scales, rows, k, kp, out, ld, stream);
}

// x += delta (where delta is not null); codes, scales = x / sqrt(mean(x^2) + eps) * weight
extern "C" int ti_mx_rmsnorm(float* x, long long ldx, const void* delta, int delta_code, long long ldd, const float* weight,
                             int rows, int k, int kp, float eps, int bits, void* codes, void* scales, void* stream) {
    if (int rc = check_format("mx_rmsnorm", rows, k, kp, bits, codes, scales)) return rc;
    TI_REQUIRE(delta_code == TI_F32 || delta_code == TI_BF16, "mx_rmsnorm: dtype code %d", delta_code);
    if (rows == 0) return 0;
    auto run = delta_code == TI_BF16 ? (bits == 8 ? rmsnorm<bf16, 8> : rmsnorm<bf16, 4>)
                                     : (bits == 8 ? rmsnorm<float, 8> : rmsnorm<float, 4>);
    return run(x, ldx, delta, ldd, weight, rows, k, kp, eps, codes, scales, stream);
}
