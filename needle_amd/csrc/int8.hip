// Rows in 8-bit integers with a scale each, and their products.
//
//   quantize:  s_i = max_j |x_ij| * (1/127),   c_ij = nearest whole number to x_ij / s_i
//   product:   out_ij = (sum_k a_ik b_jk) sa_i sb_j + bias_j
//
// The sums are exact: 32-bit integers from the matrix cores, in any order.
#include "nh_values.h"

namespace nh {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------
// quantization of rows
// ---------------------------------------------------------------------------
// The code is defined by the EXACT quotient x / s, which an f32 division can round onto a half that it is not.  So: r =
// the whole number nearest to x * (1 / s), at most one off; the residue x - r s is exact in one fused multiply-add
// (r s has at most 31 significant bits and the difference is at most about s), and it says whether r has to move:
// |residue| > s / 2, or = s / 2 with r odd.  Six instructions where the division takes a dozen.
__device__ inline int code_of(float x, float s, float inv) {
    float r = rintf(x * inv);
    const float e = __builtin_fmaf(-r, s, x), twice = 2.0f * fabsf(e);
    if (twice > s || (twice == s && ((int)r & 1))) r += e > 0.0f ? 1.0f : -1.0f;
    return (int)fminf(fmaxf(r, -127.0f), 127.0f);
}
// Rows of tiny values are scaled up by a power of two first (exact): neither 1 / s nor the residue may leave the range
// in which f32 is exact.
constexpr float PER_STEP = 1.0f / 127.0f;  // the f32 nearest to it
constexpr float TINY_ROW = 0x1p-60f, TINY_UP = 0x1p80f;

template <typename V>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const typename V::bits* __restrict__ x, uint64_t n, uint32_t dim,
                                                            uint64_t x_stride, int8_t* __restrict__ codes, uint64_t c_stride,
                                                            float* __restrict__ scales) {
    const uint32_t lane = threadIdx.x & 63;
    for (uint64_t row = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < n; row += (uint64_t)gridDim.x * 4) {
        const typename V::bits* p = x + row * x_stride;
        int8_t* c = codes + row * c_stride;
        uint32_t top = 0;  // |x| as bits: ordered like the values, NaN and infinity on top
        for (uint32_t j = lane; j < dim; j += 64) top = max(top, __float_as_uint(V::widen(p[j])) & 0x7fffffffu);
        for (int o = 32; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
        const float big = __uint_as_float(top), s = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : big * PER_STEP;
        if (lane == 0) scales[row] = s;
        if (!(s > 0.0f)) {
            for (uint32_t j = lane; j < dim; j += 64) c[j] = 0;
        } else {
            const float up = big < TINY_ROW ? TINY_UP : 1.0f, su = s * up, inv = 1.0f / su;
            for (uint32_t j = lane; j < dim; j += 64) c[j] = (int8_t)code_of(V::widen(p[j]) * up, su, inv);
        }
    }
}

// Flags rows with a NaN scale (the host form refuses them).
__global__ void nan_scales_kernel(const float* __restrict__ scales, uint64_t n, uint32_t* __restrict__ found) {
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (uint64_t)gridDim.x * blockDim.x)
        if (scales[i] != scales[i]) atomicOr(found, 1u);
}
__global__ void clear_word_kernel(uint32_t* p) { *p = 0; }

static hipError_t launch_quantize_rows(const void* x, int value, uint64_t n, uint32_t dim, uint64_t x_stride, int8_t* codes,
                                       uint64_t c_stride, float* scales, hipStream_t stream) {
    const dim3 grid((uint32_t)std::min<uint64_t>((n + 3) / 4, 1u << 20));
    switch (value) {
    case NEEDLE_VALUE_F32:
        hipLaunchKernelGGL((quantize_rows_kernel<ValueF32>), grid, dim3(256), 0, stream, (const uint32_t*)x, n, dim, x_stride, codes, c_stride, scales);
        break;
    case NEEDLE_VALUE_F16:
        hipLaunchKernelGGL((quantize_rows_kernel<ValueF16>), grid, dim3(256), 0, stream, (const uint16_t*)x, n, dim, x_stride, codes, c_stride, scales);
        break;
    default:
        hipLaunchKernelGGL((quantize_rows_kernel<ValueBF16>), grid, dim3(256), 0, stream, (const uint16_t*)x, n, dim, x_stride, codes, c_stride, scales);
    }
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------
struct MatmulParams {
    const int8_t* a;  // [m] rows, a_stride apart: queries or tokens
    const int8_t* b;  // [n] rows: base rows or output channels
    const float* a_scales;
    const float* b_scales;
    const float* bias;  // [n] or null
    void* out;
    uint64_t a_stride, b_stride, out_stride, n;
    uint32_t m, k;
};

// 16 codes of a row from place `at` on, zero from k on; nothing outside the row is read.
__device__ inline u32x4 load_codes(const int8_t* row, uint32_t at, uint32_t k) {
    if (at + 16 <= k) return *(const u32x4_any*)(row + at);
    uint32_t w[4] = {0, 0, 0, 0};
    for (uint32_t j = 0; at + j < k; ++j) w[j >> 2] |= (uint32_t)(uint8_t)row[at + j] << (8 * (j & 3));
    return u32x4{w[0], w[1], w[2], w[3]};
}

// Any sizes, strides and alignment.  A workgroup makes 64 rows of b x 64 rows of a: both pass through LDS in slices of
// 64 codes (rows of 80 bytes: the 16-byte reads of a quarter wave meet every bank once).  The rows of b are the matrix
// instruction's rows, so a lane ends up with four neighbouring outputs of one row of `out`.
template <typename V>
__global__ __launch_bounds__(256) void matmul_i8_kernel(MatmulParams p) {
    __shared__ __align__(16) uint8_t s_b[64][80], s_a[64][80];
    const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6, l15 = lane & 15, quad = lane >> 4;
    const uint64_t tiles_n = (p.n + 63) / 64, tiles = tiles_n * ((p.m + 63) / 64);
    for (uint64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const uint64_t n0 = tile % tiles_n * 64;
        const uint32_t m0 = (uint32_t)(tile / tiles_n) * 64;
        const uint32_t r = t >> 2, ch = (t & 3) * 16;
        const int8_t* rb = p.b + min(n0 + r, p.n - 1) * p.b_stride;  // rows behind the last: a copy of it, never stored
        const int8_t* ra = p.a + (uint64_t)min(m0 + r, p.m - 1) * p.a_stride;
        i32x4 acc[4] = {};
        for (uint32_t k0 = 0; k0 < p.k; k0 += 64) {
            const u32x4 vb = load_codes(rb, k0 + ch, p.k), va = load_codes(ra, k0 + ch, p.k);
            __syncthreads();
            *(u32x4*)&s_b[r][ch] = vb;
            *(u32x4*)&s_a[r][ch] = va;
            __syncthreads();
            const i32x4 fb = *(const i32x4*)&s_b[wave * 16 + l15][quad * 16];
#pragma unroll
            for (int q = 0; q < 4; ++q)
                acc[q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb, *(const i32x4*)&s_a[q * 16 + l15][quad * 16], acc[q], 0, 0, 0);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t i = m0 + q * 16 + l15;
            const uint64_t j0 = n0 + wave * 16 + quad * 4;
            if (i >= p.m) continue;
            const float sa = p.a_scales[i];
            typename V::bits* o = (typename V::bits*)p.out + (uint64_t)i * p.out_stride;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (j0 + e >= p.n) break;
                float y = (float)acc[q][e] * sa * p.b_scales[j0 + e];
                if (p.bias) y += p.bias[j0 + e];
                o[j0 + e] = V::round(y);
            }
        }
    }
}

static hipError_t launch_matmul_i8(const MatmulParams& p, int out_value, hipStream_t stream) {
    const uint64_t tiles = ((p.n + 63) / 64) * ((p.m + 63) / 64);
    const dim3 grid((uint32_t)std::min<uint64_t>(tiles, 1u << 22));
    switch (out_value) {
    case NEEDLE_VALUE_F32: hipLaunchKernelGGL((matmul_i8_kernel<ValueF32>), grid, dim3(256), 0, stream, p); break;
    case NEEDLE_VALUE_F16: hipLaunchKernelGGL((matmul_i8_kernel<ValueF16>), grid, dim3(256), 0, stream, p); break;
    default: hipLaunchKernelGGL((matmul_i8_kernel<ValueBF16>), grid, dim3(256), 0, stream, p);
    }
    return hipGetLastError();
}

constexpr uint32_t I8_K_MAX = 131071;  // 2^14 per product at most, sums below 2^31

static needle_hip_status quantize_check(needle_hip_ctx* c, const void* rows, int value, uint64_t n, uint32_t dim, uint64_t row_stride,
                                        const int8_t* codes, uint64_t code_stride, const float* scales) {
    if (!c) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "ctx is null");
    if (!value_known(value)) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "unknown value type %d", value);
    if (n == 0) return NEEDLE_HIP_OK;
    if (!scales || (dim > 0 && (!rows || !codes))) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "null argument");
    if (n > 1 && (row_stride < dim || code_stride < dim))
        return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "a stride is smaller than the %u elements of a row", dim);
    uint64_t in, out;
    if (n > (1ull << 40) || !span_bytes(n, dim, row_stride, value_size(value), &in) || !span_bytes(n, dim, code_stride, 1, &out))
        return fail(NEEDLE_HIP_ERR_UNSUPPORTED, "the rows span more than 2^62 bytes");
    if ((uintptr_t)rows % value_size(value) || (uintptr_t)scales % 4)
        return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "a pointer is not aligned to its element");
    if (ranges_meet(rows, in, codes, out) || ranges_meet(rows, in, scales, n * 4) || ranges_meet(codes, out, scales, n * 4))
        return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "an output overlaps another array");
    return NEEDLE_HIP_OK;
}

static needle_hip_status matmul_check(needle_hip_ctx* c, const void* a, uint32_t a_size, uint64_t a_stride, const float* a_scales, bool own_scales, uint32_t m,
                                      const int8_t* b, uint64_t b_stride, const float* b_scales, uint64_t n, uint32_t k,
                                      const float* bias, int out_value, const void* out, uint64_t out_stride) {
    if (!c) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "ctx is null");
    if (!value_known(out_value)) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "unknown value type %d", out_value);
    if (k > I8_K_MAX) return fail(NEEDLE_HIP_ERR_UNSUPPORTED, "k = %u exceeds %u: a sum could leave 32 bits", k, I8_K_MAX);
    if (n >= (1ull << 31)) return fail(NEEDLE_HIP_ERR_UNSUPPORTED, "at most 2^31-1 rows of b");
    if (m == 0 || n == 0) return NEEDLE_HIP_OK;
    if ((!a_scales && !own_scales) || !b_scales || !out || (k > 0 && (!a || !b))) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "null argument");
    if ((m > 1 && (a_stride < k || out_stride < n)) || (n > 1 && b_stride < k))
        return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "a stride is smaller than its row");
    uint64_t na, nb, no;
    if (!span_bytes(m, k, a_stride, a_size, &na) || !span_bytes(n, k, b_stride, 1, &nb) ||
        !span_bytes(m, n, out_stride, value_size(out_value), &no))
        return fail(NEEDLE_HIP_ERR_UNSUPPORTED, "an array spans more than 2^62 bytes");
    if ((uintptr_t)a % a_size || (uintptr_t)a_scales % 4 || (uintptr_t)b_scales % 4 || (uintptr_t)bias % 4 || (uintptr_t)out % value_size(out_value))
        return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "a pointer is not aligned to its element");
    if (ranges_meet(out, no, a, na) || ranges_meet(out, no, b, nb) || ranges_meet(out, no, a_scales, (uint64_t)m * 4) ||
        ranges_meet(out, no, b_scales, n * 4) || ranges_meet(out, no, bias, n * 4))
        return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "the output overlaps an input");
    return NEEDLE_HIP_OK;
}

}  // namespace nh

using namespace nh;

extern "C" needle_hip_status needle_hip_quantize_rows_i8_device(needle_hip_ctx* c, const void* d_rows, int value, uint64_t n, uint32_t dim,
                                                                uint64_t row_stride, int8_t* d_out_codes, uint64_t code_stride,
                                                                float* d_out_scales) {
    ST_TRY(quantize_check(c, d_rows, value, n, dim, row_stride, d_out_codes, code_stride, d_out_scales));
    if (n == 0) return NEEDLE_HIP_OK;
    std::lock_guard g(c->mu);
    DeviceScope dev(c->device);
    HIP_TRY(dev.error());
    HIP_TRY(launch_quantize_rows(d_rows, value, n, dim, row_stride, d_out_codes, code_stride, d_out_scales, c->stream));
    HIP_TRY(hipStreamSynchronize(c->stream));
    return NEEDLE_HIP_OK;
}

extern "C" needle_hip_status needle_hip_quantize_rows_i8(needle_hip_ctx* c, const void* rows, int value, uint64_t n, uint32_t dim,
                                                         int8_t* out_codes, float* out_scales) {
    ST_TRY(quantize_check(c, rows, value, n, dim, dim, out_codes, dim, out_scales));
    if (n == 0) return NEEDLE_HIP_OK;
    std::lock_guard g(c->mu);
    DeviceScope dev(c->device);
    HIP_TRY(dev.error());
    const size_t in = ((size_t)n * dim * value_size(value) + 15) & ~(size_t)15, sc = ((size_t)n * 4 + 15) & ~(size_t)15;
    HIP_TRY(c->scratch[2].ensure(in + sc + 16 + (size_t)n * dim));
    unsigned char* d = c->scratch[2].as<unsigned char>();
    float* d_scales = (float*)(d + in);
    uint32_t* d_found = (uint32_t*)(d + in + sc);
    int8_t* d_codes = (int8_t*)(d + in + sc + 16);
    if (dim) HIP_TRY(hipMemcpyAsync(d, rows, (size_t)n * dim * value_size(value), hipMemcpyHostToDevice, c->stream));
    HIP_TRY(launch_quantize_rows(d, value, n, dim, dim, d_codes, dim, d_scales, c->stream));
    hipLaunchKernelGGL(clear_word_kernel, dim3(1), dim3(1), 0, c->stream, d_found);
    hipLaunchKernelGGL(nan_scales_kernel, dim3((uint32_t)std::min<uint64_t>((n + 255) / 256, 4096)), dim3(256), 0, c->stream, d_scales, n, d_found);
    HIP_TRY(hipGetLastError());
    uint32_t found = 0;
    HIP_TRY(hipMemcpyAsync(&found, d_found, 4, hipMemcpyDeviceToHost, c->stream));
    HIP_TRY(hipStreamSynchronize(c->stream));
    if (found) return fail(NEEDLE_HIP_ERR_INVALID_VECTOR, "a row holds a NaN or an infinity");
    if (dim) HIP_TRY(hipMemcpyAsync(out_codes, d_codes, (size_t)n * dim, hipMemcpyDeviceToHost, c->stream));
    HIP_TRY(hipMemcpyAsync(out_scales, d_scales, (size_t)n * 4, hipMemcpyDeviceToHost, c->stream));
    HIP_TRY(hipStreamSynchronize(c->stream));
    return NEEDLE_HIP_OK;
}

extern "C" needle_hip_status needle_hip_matmul_i8_device(needle_hip_ctx* c, const int8_t* d_a, uint64_t a_stride, const float* d_a_scales,
                                                         uint32_t m, const int8_t* d_b, uint64_t b_stride, const float* d_b_scales,
                                                         uint64_t n, uint32_t k, const float* d_bias, int out_value, void* d_out,
                                                         uint64_t out_stride) {
    ST_TRY(matmul_check(c, d_a, 1, a_stride, d_a_scales, false, m, d_b, b_stride, d_b_scales, n, k, d_bias, out_value, d_out, out_stride));
    if (m == 0 || n == 0) return NEEDLE_HIP_OK;
    std::lock_guard g(c->mu);
    DeviceScope dev(c->device);
    HIP_TRY(dev.error());
    const MatmulParams p{d_a, d_b, d_a_scales, d_b_scales, d_bias, d_out, a_stride, b_stride, out_stride, n, m, k};
    HIP_TRY(launch_matmul_i8(p, out_value, c->stream));
    HIP_TRY(hipStreamSynchronize(c->stream));
    return NEEDLE_HIP_OK;
}

extern "C" needle_hip_status needle_hip_matmul_i8(needle_hip_ctx* c, const int8_t* a, const float* a_scales, uint32_t m, const int8_t* b,
                                                  const float* b_scales, uint64_t n, uint32_t k, const float* bias, float* out) {
    ST_TRY(matmul_check(c, a, 1, k, a_scales, false, m, b, k, b_scales, n, k, bias, NEEDLE_VALUE_F32, out, n));
    if (m == 0 || n == 0) return NEEDLE_HIP_OK;
    std::lock_guard g(c->mu);
    DeviceScope dev(c->device);
    HIP_TRY(dev.error());
    const size_t sizes[6] = {(size_t)m * k, (size_t)n * k, (size_t)m * 4, (size_t)n * 4, bias ? (size_t)n * 4 : 0, (size_t)m * n * 4};
    size_t at[7] = {0};
    for (int i = 0; i < 6; ++i) at[i + 1] = at[i] + ((sizes[i] + 15) & ~(size_t)15);
    HIP_TRY(c->scratch[4].ensure(at[6]));
    unsigned char* d = c->scratch[4].as<unsigned char>();
    const void* src[5] = {a, b, a_scales, b_scales, bias};
    for (int i = 0; i < 5; ++i)
        if (sizes[i]) HIP_TRY(hipMemcpyAsync(d + at[i], src[i], sizes[i], hipMemcpyHostToDevice, c->stream));
    const MatmulParams p{(const int8_t*)(d + at[0]), (const int8_t*)(d + at[1]), (const float*)(d + at[2]), (const float*)(d + at[3]),
                         bias ? (const float*)(d + at[4]) : nullptr, d + at[5], k, k, n, n, m, k};
    HIP_TRY(launch_matmul_i8(p, NEEDLE_VALUE_F32, c->stream));
    HIP_TRY(hipMemcpyAsync(out, d + at[5], sizes[5], hipMemcpyDeviceToHost, c->stream));
    HIP_TRY(hipStreamSynchronize(c->stream));
    return NEEDLE_HIP_OK;
}

extern "C" needle_hip_status needle_hip_linear_i8_device(needle_hip_ctx* c, const void* d_x, int x_value, uint64_t x_stride, uint32_t m,
                                                         const int8_t* d_b, uint64_t b_stride, const float* d_b_scales, uint64_t n,
                                                         uint32_t k, const float* d_bias, int out_value, void* d_out, uint64_t out_stride) {
    if (!value_known(x_value)) return fail(NEEDLE_HIP_ERR_INVALID_ARGUMENT, "unknown value type %d", x_value);
    ST_TRY(matmul_check(c, d_x, value_size(x_value), x_stride, nullptr, true, m, d_b, b_stride, d_b_scales, n, k, d_bias, out_value, d_out,
                        out_stride));
    if (m == 0 || n == 0) return NEEDLE_HIP_OK;
    std::lock_guard g(c->mu);
    DeviceScope dev(c->device);
    HIP_TRY(dev.error());
    const uint64_t stride = ((uint64_t)k + 127) / 128 * 128;
    HIP_TRY(c->scratch[6].ensure((size_t)m * stride + (size_t)m * 4));
    int8_t* d_codes = c->scratch[6].as<int8_t>();
    float* d_scales = (float*)(d_codes + (size_t)m * stride);
    HIP_TRY(launch_quantize_rows(d_x, x_value, m, k, x_stride, d_codes, stride, d_scales, c->stream));
    const MatmulParams p{d_codes, d_b, d_scales, d_b_scales, d_bias, d_out, stride, b_stride, out_stride, n, m, k};
    HIP_TRY(launch_matmul_i8(p, out_value, c->stream));
    HIP_TRY(hipStreamSynchronize(c->stream));
    return NEEDLE_HIP_OK;
}
