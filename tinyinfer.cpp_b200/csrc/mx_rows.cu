// Rows into the microscaled format (mx.cuh), out of it, and the root-mean-square norm whose output is in it.
//
// All three are bound by the bytes they move and, for few rows, by one round trip to memory; the first two come close to the
// limit of instructions too, so a thread's place costs no division (a block is a power of two of threads along a row) and
// conversions are the hardware's, two elements each.  A thread owns eight neighbouring elements at a time (16 bytes of
// bfloat16, 32 of float32), so a block of 32 is four lanes and a chunk of 128 sixteen: the block's largest magnitude is two
// shuffles, a chunk's four scale bytes meet in one lane, which stores them as a word.  Rows whose start, stride or length does
// not allow such accesses are read element by element (the lines come from L1) and written by warps that walk a chunk with
// one element of each of its blocks a lane.
#include <cuda_fp16.h>

#include "mx.cuh"

namespace {

using namespace mx;

constexpr int UNIT = 8;                 // elements of a thread

// The next kernel's blocks may come while these run, unless there are more of these than SMs: they would take the places of the
// ones that wait (norm with a delta, 4,096 x 512: 6.4 us with, 5.3 without; 8 rows: a product behind starts earlier).
__device__ __forceinline__ void launch_next_early() {
    if ((long long)gridDim.x * gridDim.y <= 148) pdl_launch();
}

__device__ __forceinline__ void widen(const uint4& raw, float (&v)[UNIT]) {
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void load_unit(const bf16* p, float (&v)[UNIT]) { widen(*reinterpret_cast<const uint4*>(p), v); }
__device__ __forceinline__ void load_unit(const float* p, float (&v)[UNIT]) {
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

// The largest magnitude's float32 bits, over the thread's elements and over its block's.  Bits, not numbers: a NaN is larger
// than everything then.
__device__ __forceinline__ unsigned top_of_block(unsigned top) {
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    return max(top, __shfl_xor_sync(0xffffffffu, top, 2));
}
__device__ __forceinline__ unsigned top_of(const float (&v)[UNIT]) {
    unsigned b[UNIT];
#pragma unroll
    for (int i = 0; i < UNIT; ++i) b[i] = __float_as_uint(v[i]) & 0x7fffffffu;
    const unsigned x = __vimax3_u32(b[0], b[1], b[2]), y = __vimax3_u32(b[3], b[4], b[5]);
    return top_of_block(max(__vimax3_u32(x, y, b[6]), b[7]));
}
// ... of eight bfloat16 as they were loaded: two at a time
__device__ __forceinline__ unsigned top_of(const uint4& raw) {
    unsigned t = __vmaxu2(__vmaxu2(raw.x & 0x7fff7fffu, raw.y & 0x7fff7fffu), __vmaxu2(raw.z & 0x7fff7fffu, raw.w & 0x7fff7fffu));
    t = __vmaxu2(t, __shfl_xor_sync(0xffffffffu, t, 1));
    t = __vmaxu2(t, __shfl_xor_sync(0xffffffffu, t, 2));
    return max(t & 0xffff0000u, t << 16);
}

// Codes and scales of a thread's eight elements at column c of a row, `top` their block's largest magnitude, c a multiple of
// 128 in the first of sixteen lanes.  A whole warp calls it (shuffles under a mask that is not known when compiling cost far
// more), lanes with nothing to store with `valid` false.  `at`, `scale_words`: where the row's codes and the scale words of its
// chunks begin (a row's words are 512 bytes apart).
template <int BITS>
__device__ __forceinline__ void store_codes(const float (&v)[UNIT], unsigned top, int c, bool valid, unsigned char* at,
                                            unsigned char* scale_words) {
    const unsigned s = scale_byte<BITS>(top);
    const float inv = scale_inverse(s);
    float y[UNIT];
#pragma unroll
    for (int i = 0; i < UNIT; ++i) y[i] = v[i] * inv;
    if (BITS == 8) {
        const uint2 w = make_uint2(codes_e4m3x4(y), codes_e4m3x4(y + 4));
        if (valid) *reinterpret_cast<uint2*>(at + c) = w;
    } else {
        const unsigned w = codes_e2m1x8(y);
        if (valid) *reinterpret_cast<unsigned*>(at + c / 2) = w;
    }
    unsigned word = s << (8 * (threadIdx.x >> 2 & 3));       // the four blocks of a chunk: lanes 0, 4, 8, 12 of sixteen
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    if (valid && (threadIdx.x & 15) == 0) *reinterpret_cast<unsigned*>(scale_words + (size_t)(c / CHUNK) * TILE_BYTES) = word;
}

// ---- quantisation --------------------------------------------------------------------------------

constexpr int QUANT_THREADS = 256;

// Where a thread of a row kernel works: 1 << shift threads lie along a row, QUANT_THREADS >> shift rows are in a block, and
// blockIdx.y counts segments of `ahead` << shift units of a row, `ahead` of them a thread's, all asked for before the first
// is used.
struct Place {
    long long row;
    int unit;                           // the first; the others follow at distances of 1 << shift
    __device__ Place(int shift, int ahead)
        : row(((long long)blockIdx.x << (8 - shift)) + (threadIdx.x >> shift)),
          unit((int)((blockIdx.y * ahead) << shift) + ((int)threadIdx.x & ((1 << shift) - 1))) {}
};

// Eight elements as they were loaded, then as numbers with their block's top.  `held` of them are inside the row; WHOLE: all
// or none, on 16 bytes.
template <typename T, bool WHOLE> struct Unit {
    float v[UNIT];
    __device__ void load(const T* p, int held) {
        if (WHOLE) {
            if (held > 0) {
                load_unit(p, v);
                return;
            }
            held = 0;
        }
#pragma unroll
        for (int i = 0; i < UNIT; ++i) v[i] = i < held ? to_f32(p[i]) : 0.0f;
    }
    __device__ unsigned take(float (&out)[UNIT]) const {
#pragma unroll
        for (int i = 0; i < UNIT; ++i) out[i] = v[i];
        return top_of(v);
    }
};
template <> struct Unit<bf16, true> {
    uint4 raw;
    __device__ void load(const bf16* p, int held) {
        raw = held > 0 ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
    }
    __device__ unsigned take(float (&out)[UNIT]) const {
        widen(raw, out);
        return top_of(raw);
    }
};

template <typename T, int BITS, bool WHOLE, int AHEAD>
__global__ void __launch_bounds__(QUANT_THREADS)
mx_quantize_kernel(const T* x, long long ld, int rows, int k, int kp, unsigned char* codes, unsigned char* scales, int shift) {
    const Place me(shift, AHEAD);
    launch_next_early();
    pdl_wait();
    const T* from = x + (size_t)me.row * ld;
    Unit<T, WHOLE> units[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
        const int c = (me.unit + (u << shift)) * UNIT;
        units[u].load(from + c, me.row < rows ? k - c : 0);
    }
    unsigned char *at = codes + (size_t)me.row * kp / (8 / BITS), *words = scales + scale_at((int)me.row, 0, kp / CHUNK);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
        const int c = (me.unit + (u << shift)) * UNIT;
        float v[UNIT];
        const unsigned top = units[u].take(v);
        store_codes<BITS>(v, top, c, me.row < rows && c < kp, at, words);
    }
}

// ---- and back ------------------------------------------------------------------------------------

// two codes as numbers without their scale (both element types are exact in float16), one, eight
template <int BITS> __device__ __forceinline__ __half2 values_of2(unsigned codes) {
    unsigned pair;
    if (BITS == 8)
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(pair) : "h"((unsigned short)codes));
    else
        asm("{\n\t.reg .b8 b;\n\tcvt.u8.u32 b, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(pair) : "r"(codes));
    return *reinterpret_cast<const __half2*>(&pair);
}
template <int BITS> __device__ __forceinline__ float value_of(unsigned code) { return __low2float(values_of2<BITS>(code)); }
template <int BITS> __device__ __forceinline__ void values_of(uint2 w, float (&v)[UNIT]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(values_of2<BITS>(BITS == 8 ? (i < 2 ? w.x : w.y) >> (16 * (i & 1)) : w.x >> (8 * i)));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

template <typename T, int BITS, int AHEAD>
__global__ void __launch_bounds__(QUANT_THREADS)
mx_dequantize_kernel(const unsigned char* codes, const unsigned char* scales, int rows, int k, int kp, T* out, long long ld,
                     int shift) {
    const Place me(shift, AHEAD);
    launch_next_early();
    pdl_wait();
    if (me.row >= rows) return;
    const unsigned char *at = codes + (size_t)me.row * kp / (8 / BITS), *words = scales + scale_at((int)me.row, 0, kp / CHUNK);
    uint2 w[AHEAD];
    unsigned s[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
        const int c = (me.unit + (u << shift)) * UNIT;
        if (c < k) {
            w[u] = BITS == 8 ? *reinterpret_cast<const uint2*>(at + c)
                             : make_uint2(*reinterpret_cast<const unsigned*>(at + c / 2), 0);
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
        store_unit(out + (size_t)me.row * ld + c, v);         // k is a multiple of 8
    }
}

// rows of the output off 16 bytes
template <typename T, int BITS>
__global__ void __launch_bounds__(QUANT_THREADS)
mx_dequantize_any_kernel(const unsigned char* codes, const unsigned char* scales, int rows, int k, int kp, T* out, long long ld,
                         int) {
    const unsigned chunks = (unsigned)kp / CHUNK, at = (blockIdx.x * QUANT_THREADS + threadIdx.x) / 32;
    const int lane = threadIdx.x & 31;
    launch_next_early();
    pdl_wait();
    if (at >= (unsigned)rows * chunks) return;
    const int row = (int)(at / chunks), c = (int)(at % chunks) * CHUNK;
    const unsigned word = *reinterpret_cast<const unsigned*>(scales + scale_at(row, c / BLOCK, kp / CHUNK));
    const unsigned char* from = codes + ((size_t)row * kp + c) / (8 / BITS);
    T* to = out + (size_t)row * ld + c;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const int e = b * BLOCK + lane;
        const unsigned code = BITS == 8 ? from[e] : from[e / 2] >> (4 * (lane & 1));      // above a code is its neighbour
        const float v = value_of<BITS>(code) * scale_value(word >> (8 * b) & 255u);
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
    launch_next_early();
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
        float w[UNIT];
        load_guarded(weight, c, k, whole_w, w);
#pragma unroll
        for (int i = 0; i < UNIT; ++i) v[u][i] = v[u][i] * inv * w[i];
        store_codes<BITS>(v[u], top_of(v[u]), c, c < kp, codes + (size_t)row * kp / (8 / BITS),
                          scales + scale_at(row, 0, kp / CHUNK));
    }
}

bool whole_rows(const void* p, long long ld, int bytes) { return (uintptr_t)p % 16 == 0 && ld * bytes % 16 == 0; }

// The launch of a row kernel over `units` of eight elements a row: as many threads along a row as its units want (16 to 256).
// Four units a thread where the GPU (148 SMs of 2,048 threads) is full all the same, else one: 12,288 x 4,096 bfloat16 into 4
// bits and back 31.7 + 30.9 us with one, 27.0 + 23.5 with two, 24.0 + 21.2 with four; 8 x 4,096 1.38 us with one, 1.85 with two.
struct Shape {
    dim3 grid;
    int shift = 8, ahead;
    Shape(long long rows, int units) : ahead(rows * units >= 4LL * 148 * 2048 ? 4 : 1) {
        while (shift > 4 && ahead << (shift - 1) >= units) --shift;
        const long long in_block = QUANT_THREADS >> shift, segments = (units + (ahead << shift) - 1) / (ahead << shift);
        grid = dim3((unsigned)((rows + in_block - 1) / in_block), (unsigned)segments);
    }
};

template <typename T, int BITS>
int quantize(const void* x, long long ld, int rows, int k, int kp, void* codes, void* scales, void* stream) {
    const bool whole = whole_rows(x, ld, sizeof(T)) && k % UNIT == 0;
    const Shape shape(rows, kp / UNIT);
    TI_REQUIRE(shape.grid.y < 65536, "mx_quantize: rows of %d elements are too long", k);
    auto kernel = shape.ahead == 4 ? (whole ? mx_quantize_kernel<T, BITS, true, 4> : mx_quantize_kernel<T, BITS, false, 4>)
                                   : (whole ? mx_quantize_kernel<T, BITS, true, 1> : mx_quantize_kernel<T, BITS, false, 1>);
    ti_launch_pdl(kernel, shape.grid, QUANT_THREADS, 0, (cudaStream_t)stream, (const T*)x, ld, rows, k, kp, (unsigned char*)codes,
                  (unsigned char*)scales, shape.shift);
    return ti_check_launch("mx_quantize");
}

template <typename T, int BITS>
int dequantize(const void* codes, const void* scales, int rows, int k, int kp, void* out, long long ld, void* stream) {
    const bool whole = whole_rows(out, ld, sizeof(T)) && k % UNIT == 0;
    Shape shape(rows, (k + UNIT - 1) / UNIT);
    auto kernel = shape.ahead == 4 ? mx_dequantize_kernel<T, BITS, 4> : mx_dequantize_kernel<T, BITS, 1>;
    if (!whole) {                                            // a warp a chunk
        const long long warps = (long long)rows * (kp / CHUNK);
        TI_REQUIRE(warps < (1LL << 27), "mx_dequantize: %d rows of %d elements are too many", rows, k);
        shape.grid = dim3((unsigned)((warps + QUANT_THREADS / 32 - 1) / (QUANT_THREADS / 32)));
        kernel = mx_dequantize_any_kernel<T, BITS>;
    }
    TI_REQUIRE(shape.grid.y < 65536, "mx_dequantize: rows of %d elements are too long", k);
    ti_launch_pdl(kernel, shape.grid, QUANT_THREADS, 0, (cudaStream_t)stream, (const unsigned char*)codes,
                  (const unsigned char*)scales, rows, k, kp, (T*)out, ld, shape.shift);
    return ti_check_launch("mx_dequantize");
}

template <typename D, int BITS>
int rmsnorm(void* x, long long ldx, const void* delta, long long ldd, const void* weight, int rows, int k, int kp, float eps,
            void* codes, void* scales, void* stream) {
    const int units = kp / UNIT;
    // As many threads as a block may have before a thread takes a second unit (us with one, two and four, with a delta: 8 x 4,096
    // 2.4, 2.8, 3.9; 4,096 x 8,192 66.9, 72.3, 73.7), except where many rows come without a delta: then 256 threads, so that
    // more rows are on the way at once (4,096 x 4,096 18.9, 17.3, 17.5; 4,096 x 8,192 41.2, 38.6, 32.5; 8 x 4,096 2.0, 2.3, 2.9).
    const int most = delta == nullptr && rows > 4 * 148 ? 256 : 1024;
    const int per = units <= most ? 1 : units <= 2 * most ? 2 : 4;
    const int threads = ((units + per - 1) / per + 31) / 32 * 32;
    TI_REQUIRE(threads <= 1024, "mx_rmsnorm: rows of %d elements are longer than 32,768", k);
    auto kernel = per == 1 ? mx_rmsnorm_kernel<D, BITS, 1>
                : per == 2 ? mx_rmsnorm_kernel<D, BITS, 2> : mx_rmsnorm_kernel<D, BITS, 4>;
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
