// Rows into the microscaled format (mx.cuh), out of it, and the root-mean-square norm whose output is in it.
//
// All three are bound by the bytes they move and, for few rows, by one round trip to memory.  A thread owns eight
// neighbouring elements (16 bytes of bfloat16, 32 of float32), so a block of 32 is four lanes and a chunk of 128 sixteen:
// the block's largest magnitude is two shuffles, a chunk's four scale bytes meet in one lane, which stores them as a word.
// Rows whose start or stride does not allow such loads take a second form in which a warp walks a block with one element a
// lane: every load is still 32 neighbours, the maximum is one redux.
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

// Codes and scales of a thread's eight elements at column c of a row; whole groups of sixteen neighbouring lanes call it
// together, c a multiple of 128 in the group's first lane.
template <int BITS>
__device__ __forceinline__ void store_codes(const float (&v)[UNIT], int row, int c, int kp, unsigned char* codes,
                                            unsigned char* scales) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < UNIT; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    const unsigned half = 0xffffu << (threadIdx.x & 16);
    top = max(top, __shfl_xor_sync(half, top, 1));
    top = max(top, __shfl_xor_sync(half, top, 2));
    const unsigned s = scale_byte<BITS>(top);
    const float inv = scale_inverse(s);
    unsigned char* at = codes + ((size_t)row * kp + c) / (8 / BITS);
    if (BITS == 8) {
        unsigned w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = codes_e4m3x2(v[4 * i] * inv, v[4 * i + 1] * inv) | codes_e4m3x2(v[4 * i + 2] * inv, v[4 * i + 3] * inv) << 16;
        *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
    } else {
        unsigned w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= codes_e2m1x2(v[2 * i] * inv, v[2 * i + 1] * inv) << (8 * i);
        *reinterpret_cast<unsigned*>(at) = w;
    }
    unsigned word = s << (8 * (threadIdx.x >> 2 & 3));       // the four blocks of a chunk: lanes 0, 4, 8, 12 of sixteen
    word |= __shfl_xor_sync(half, word, 4);
    word |= __shfl_xor_sync(half, word, 8);
    if ((threadIdx.x & 15) == 0) *reinterpret_cast<unsigned*>(scales + scale_at(row, c / BLOCK, kp / CHUNK)) = word;
}

// ---- quantisation --------------------------------------------------------------------------------

constexpr int QUANT_THREADS = 256;

template <typename T, int BITS>
__global__ void __launch_bounds__(QUANT_THREADS)
mx_quantize_kernel(const T* x, long long ld, int rows, int k, int kp, unsigned char* codes, unsigned char* scales) {
    const unsigned per_row = (unsigned)kp / UNIT, at = blockIdx.x * QUANT_THREADS + threadIdx.x;
    pdl_wait();
    if (at >= (unsigned)rows * per_row) return;              // whole groups of sixteen lanes: per_row is a multiple of 16
    const int row = (int)(at / per_row), c = (int)(at % per_row) * UNIT;
    float v[UNIT];
    load_guarded(x + (size_t)row * ld, c, k, true, v);
    store_codes<BITS>(v, row, c, kp, codes, scales);
}

// any start and stride: a warp takes a chunk, one element of each of its four blocks a lane
template <typename T, int BITS>
__global__ void __launch_bounds__(QUANT_THREADS)
mx_quantize_any_kernel(const T* x, long long ld, int rows, int k, int kp, unsigned char* codes, unsigned char* scales) {
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

template <typename T, int BITS>
__global__ void __launch_bounds__(QUANT_THREADS)
mx_dequantize_kernel(const unsigned char* codes, const unsigned char* scales, int rows, int k, int kp, T* out, long long ld,
                     bool whole) {
    const unsigned per_row = ((unsigned)k + UNIT - 1) / UNIT, at = blockIdx.x * QUANT_THREADS + threadIdx.x;
    pdl_launch();
    pdl_wait();
    if (at >= (unsigned)rows * per_row) return;
    const int row = (int)(at / per_row), c = (int)(at % per_row) * UNIT;
    const unsigned char* from = codes + ((size_t)row * kp + c) / (8 / BITS);
    const float f = scale_value(scales[scale_at(row, c / BLOCK, kp / CHUNK)]);
    float v[UNIT];
    if (BITS == 8) {
        const uint2 w = *reinterpret_cast<const uint2*>(from);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = value_e4m3(w.x >> (8 * i) & 255u) * f;
            v[4 + i] = value_e4m3(w.y >> (8 * i) & 255u) * f;
        }
    } else {
        const unsigned w = *reinterpret_cast<const unsigned*>(from);
#pragma unroll
        for (int i = 0; i < UNIT; ++i) v[i] = value_e2m1(w >> (4 * i) & 15u) * f;
    }
    store_guarded(out + (size_t)row * ld, c, k, whole, v);
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
        store_codes<BITS>(v[u], row, c, kp, codes, scales);
    }
}

bool whole_rows(const void* p, long long ld, int bytes) { return (uintptr_t)p % 16 == 0 && ld * bytes % 16 == 0; }

template <typename T, int BITS>
int quantize(const void* x, long long ld, int rows, int k, int kp, void* codes, void* scales, void* stream) {
    const bool whole = whole_rows(x, ld, sizeof(T));
    const long long threads = whole ? (long long)rows * (kp / UNIT) : (long long)rows * (kp / CHUNK) * 32;
    TI_REQUIRE(threads < (1LL << 32) - QUANT_THREADS, "mx_quantize: %d rows of %d elements are too many", rows, k);
    const unsigned blocks = (unsigned)((threads + QUANT_THREADS - 1) / QUANT_THREADS);
    ti_launch_pdl(whole ? mx_quantize_kernel<T, BITS> : mx_quantize_any_kernel<T, BITS>, blocks, QUANT_THREADS, 0,
                  (cudaStream_t)stream, (const T*)x, ld, rows, k, kp, (unsigned char*)codes, (unsigned char*)scales);
    return ti_check_launch("mx_quantize");
}

template <typename T, int BITS>
int dequantize(const void* codes, const void* scales, int rows, int k, int kp, void* out, long long ld, void* stream) {
    const long long threads = (long long)rows * ((k + UNIT - 1) / UNIT);
    TI_REQUIRE(threads < (1LL << 32) - QUANT_THREADS, "mx_dequantize: %d rows of %d elements are too many", rows, k);
    ti_launch_pdl(mx_dequantize_kernel<T, BITS>, (unsigned)((threads + QUANT_THREADS - 1) / QUANT_THREADS), QUANT_THREADS, 0,
                  (cudaStream_t)stream, (const unsigned char*)codes, (const unsigned char*)scales, rows, k, kp, (T*)out, ld,
                  whole_rows(out, ld, sizeof(T)));
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
