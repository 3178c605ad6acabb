// Rows in 8-bit integers with a scale each, and their products.
//
//   quantize:  s_i = max_j |x_ij| * (1/127),   c_ij = nearest whole number to x_ij / s_i
//   product:   out_ij = (sum_k a_ik b_jk) sa_i sb_j + bias_j
//
// The sums are exact: 32-bit integers from the matrix cores, in any order.
#include "nh_values.h"
#include <chrono>

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

// LANES lanes (256: the four waves of a workgroup) hold a row in registers, PER vectors of WIDE values each, so that it is
// read once: 16 bytes per lane and load, from any address, WIDE codes per store.  Rows longer than 256 * 8 * WIDE values are
// read twice (the second time from the cache) by a workgroup of 1024.  The bytes bound it: 200003 x 384 f32 take 68 us, 5.6
// TB/s (a wave per row, a value per load, read twice: 174 us); 41593 x 1505 bf16 37 us, 5.1 TB/s (with every residue taken, a
// dozen instructions more per value, 54).
//
// Of a row that is neither tiny nor NaN most codes need no residue: x / s and x * (1 / s) differ by 127 * 2^-24 at most, so
// where the latter lies further than that from a half, its nearest whole number is the code.  Adding 1.5 * 2^23 to the
// product leaves that number in the low bits of the sum.  A wave that meets a half takes the residues of that load.
template <typename V, int LANES, int PER>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const typename V::bits* __restrict__ x, uint64_t n, uint32_t dim,
                                                            uint64_t x_stride, int8_t* __restrict__ codes, uint64_t c_stride,
                                                            float* __restrict__ scales) {
    constexpr int WIDE = 16 / V::size;
    constexpr float WHOLE = 12582912.0f, HALF = 0.49998f;
    typedef uint32_t codes_t __attribute__((ext_vector_type(WIDE / 4), aligned(1)));
    typedef typename V::bits bits_t __attribute__((ext_vector_type(WIDE)));
    const uint32_t lane = threadIdx.x % LANES;
    const uint64_t at = ((uint64_t)blockIdx.x * 256 + threadIdx.x) / LANES;
    if (LANES <= 64 && at >= n) return;
    const uint64_t row = LANES <= 64 ? at : min(at, n - 1);  // (two rows of 128 lanes share a barrier: the last one twice if need be)
    const typename V::bits* p = x + row * x_stride;
    int8_t* c = codes + row * c_stride;
    bits_t v[PER];
    bits_t tops = 0;  // |x| as bits: ordered like the values, NaN and infinity on top
    auto load = [&](uint32_t j) {
        bits_t one;
        if (j + WIDE <= dim) return __builtin_bit_cast(bits_t, *(const u32x4_any*)(p + j));
#pragma unroll
        for (int w = 0; w < WIDE; ++w) one[w] = j + w < dim ? p[j + w] : (typename V::bits)0;
        return one;
    };
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = load((i * LANES + lane) * WIDE);
#pragma unroll
    for (int i = 0; i < PER; ++i) tops = __builtin_elementwise_max(tops, v[i] & (typename V::bits)(V::size == 2 ? 0x7fff : 0x7fffffff));
    typename V::bits most = tops[0];
#pragma unroll
    for (int w = 1; w < WIDE; ++w) most = max(most, tops[w]);
    uint32_t top = __float_as_uint(V::widen(most));
#pragma unroll
    for (int o = LANES < 64 ? LANES / 2 : 32; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    if (LANES > 64) {
        __shared__ uint32_t s_top[4];
        if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = top;
        __syncthreads();
        constexpr uint32_t WAVES = LANES / 64;
        const uint32_t first = threadIdx.x / LANES * WAVES;
#pragma unroll
        for (uint32_t w = 0; w < WAVES; ++w) top = max(top, s_top[first + w]);
    }
    const float big = __uint_as_float(top), s = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : big * PER_STEP;
    if (lane == 0) scales[row] = s;
    const bool some = s > 0.0f;
    const float up = big < TINY_ROW ? TINY_UP : 1.0f, su = some ? s * up : 1.0f, inv = 1.0f / su, fast = some ? inv : 0.0f;
    const float odd = (some && big < TINY_ROW) || s != s ? 1.0f : 0.0f;  // tiny and NaN rows
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        codes_t q;
        uint32_t t[WIDE];
        float worst = odd;
#pragma unroll
        for (int w = 0; w < WIDE; ++w) {
            const float y = V::widen(v[i][w]), whole = __builtin_fmaf(y, fast, WHOLE);
            worst = fmaxf(worst, fabsf(__builtin_fmaf(y, fast, -(whole - WHOLE))));
            t[w] = __float_as_uint(whole);
        }
        if (__any(worst > HALF)) {
#pragma unroll
            for (int w = 0; w < WIDE; ++w) t[w] = (uint32_t)(some ? code_of(V::widen(v[i][w]) * up, su, inv) : 0);
        }
#pragma unroll
        for (int w = 0; w < WIDE; w += 4)  // the low bytes
            q[w / 4] = __builtin_amdgcn_perm(t[w + 1], t[w], 0x0c0c0400u) | __builtin_amdgcn_perm(t[w + 3], t[w + 2], 0x04000c0cu);
        const uint32_t j = (i * LANES + lane) * WIDE;
        if (j + WIDE <= dim) {
            *(codes_t*)(c + j) = q;
        } else {
#pragma unroll
            for (int w = 0; w < WIDE; ++w)
                if (j + w < dim) c[j + w] = (int8_t)t[w];
        }
    }
}

template <typename V>
__global__ __launch_bounds__(1024) void quantize_long_rows_kernel(const typename V::bits* __restrict__ x, uint64_t n, uint32_t dim,
                                                                  uint64_t x_stride, int8_t* __restrict__ codes, uint64_t c_stride,
                                                                  float* __restrict__ scales) {
    constexpr uint32_t WIDE = 16 / V::size, AT_ONCE = 1024 * WIDE;
    typedef int8_t codes_t __attribute__((ext_vector_type(WIDE), aligned(1)));
    __shared__ uint32_t s_top[16];
    const uint32_t t = threadIdx.x;
    for (uint64_t row = blockIdx.x; row < n; row += gridDim.x) {
        const typename V::bits* p = x + row * x_stride;
        int8_t* c = codes + row * c_stride;
        const uint32_t whole = dim / WIDE * WIDE, left = dim - whole;
        uint32_t top = 0;
        for (uint64_t j = t * WIDE; j < whole; j += AT_ONCE) {  // (64 bits: a step past a long row's end)
            const u32x4 raw = *(const u32x4_any*)(p + j);
            typename V::bits one[WIDE];
            __builtin_memcpy(one, &raw, 16);
#pragma unroll
            for (int w = 0; w < (int)WIDE; ++w) top = max(top, __float_as_uint(V::widen(one[w])) & 0x7fffffffu);
        }
        if (t < left) top = max(top, __float_as_uint(V::widen(p[whole + t])) & 0x7fffffffu);
        for (int o = 32; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
        __syncthreads();  // (the row before has left s_top)
        if ((t & 63) == 0) s_top[t >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 16; ++w) top = max(top, s_top[w]);
        const float big = __uint_as_float(top), s = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : big * PER_STEP;
        if (t == 0) scales[row] = s;
        const bool some = s > 0.0f;
        const float up = big < TINY_ROW ? TINY_UP : 1.0f, su = some ? s * up : 1.0f, inv = 1.0f / su;
        for (uint64_t j = t * WIDE; j < whole; j += AT_ONCE) {
            const u32x4 raw = *(const u32x4_any*)(p + j);
            typename V::bits one[WIDE];
            __builtin_memcpy(one, &raw, 16);
            codes_t q;
#pragma unroll
            for (int w = 0; w < (int)WIDE; ++w) q[w] = (int8_t)(some ? code_of(V::widen(one[w]) * up, su, inv) : 0);
            *(codes_t*)(c + j) = q;
        }
        if (t < left) c[whole + t] = (int8_t)(some ? code_of(V::widen(p[whole + t]) * up, su, inv) : 0);
    }
}

// A call ends with a kernel that counts up a pinned word, which the host watches: 2 us sooner than the stream's
// synchronization after a short kernel, 3 after one of 80 us.  The kernel starts when those before it have finished and
// their writes are out.  The watch is given up for the synchronization, which sleeps and reports errors, after 1 ms.
__global__ void done_kernel(uint32_t* word, uint32_t count) { __hip_atomic_store(word, count, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM); }
hipError_t wait_done(needle_hip_ctx* c) {
    if (!c->done) {
        const hipError_t e = hipHostMalloc((void**)&c->done, 64, hipHostMallocCoherent);
        if (e != hipSuccess) {
            c->done = nullptr;
            return e;
        }
        *c->done = c->done_count;
    }
    const uint32_t count = ++c->done_count;
    hipLaunchKernelGGL(done_kernel, dim3(1), dim3(1), 0, c->stream, c->done, count);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const auto start = std::chrono::steady_clock::now();
    for (uint32_t i = 1; __atomic_load_n(c->done, __ATOMIC_ACQUIRE) != count; ++i)
        if (i % 64 == 0 && std::chrono::steady_clock::now() - start > std::chrono::milliseconds(1)) return hipStreamSynchronize(c->stream);
    return hipSuccess;
}

// Flags rows with a NaN scale (the host form refuses them).
__global__ void nan_scales_kernel(const float* __restrict__ scales, uint64_t n, uint32_t* __restrict__ found) {
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (uint64_t)gridDim.x * blockDim.x)
        if (scales[i] != scales[i]) atomicOr(found, 1u);
}
__global__ void clear_word_kernel(uint32_t* p) { *p = 0; }

template <typename V, int LANES, int PER>
static void launch_quantize_of(const typename V::bits* x, uint64_t n, uint32_t dim, uint64_t x_stride, int8_t* codes, uint64_t c_stride,
                               float* scales, hipStream_t stream) {
    constexpr uint64_t ROWS = 256 / LANES, MOST = (1u << 23) * ROWS;  // rows per workgroup and launch
    for (uint64_t r = 0; r < n; r += MOST) {
        const uint64_t rows = std::min(MOST, n - r);
        hipLaunchKernelGGL((quantize_rows_kernel<V, LANES, PER>), dim3((uint32_t)((rows + ROWS - 1) / ROWS)), dim3(256), 0, stream, x + r * x_stride, rows,
                           dim, x_stride, codes + r * c_stride, c_stride, scales + r);
    }
}
template <typename V>
static hipError_t launch_quantize_rows_of(const typename V::bits* x, uint64_t n, uint32_t dim, uint64_t x_stride, int8_t* codes, uint64_t c_stride,
                                          float* scales, hipStream_t stream) {
    const uint32_t loads = (uint32_t)(((uint64_t)dim + 16 / V::size - 1) / (16 / V::size));  // of a row
    // several loads per lane where the row has them, few idle lanes: us of 1000000 x 64 f32 with <4, 2>, <8, 1>: 56, 69 (less a
    // call's 17); 100000 x 384 f16 with <16, 3>, <32, 2>: 24, 34; 3000000 x 24 bf16 with <4, 1>, <8, 1>: 64, 128; 16384 x 4096
    // bf16 with <256, 2>, <64, 8>: 41, 44; 30000 x 1000 f32 with <64, 4>, <256, 1>: 23, 30
    if (loads <= 4) launch_quantize_of<V, 4, 1>(x, n, dim, x_stride, codes, c_stride, scales, stream);
    else if (loads <= 8) launch_quantize_of<V, 4, 2>(x, n, dim, x_stride, codes, c_stride, scales, stream);
    else if (loads <= 16) launch_quantize_of<V, 8, 2>(x, n, dim, x_stride, codes, c_stride, scales, stream);
    else if (loads <= 32) launch_quantize_of<V, 16, 2>(x, n, dim, x_stride, codes, c_stride, scales, stream);
    else if (loads <= 48) launch_quantize_of<V, 16, 3>(x, n, dim, x_stride, codes, c_stride, scales, stream);
    else if (loads <= 64) launch_quantize_of<V, 32, 2>(x, n, dim, x_stride, codes, c_stride, scales, stream);
    else if (loads <= 96) launch_quantize_of<V, 32, 3>(x, n, dim, x_stride, codes, c_stride, scales, stream);
    else if (loads <= 128) launch_quantize_of<V, 64, 2>(x, n, dim, x_stride, codes, c_stride, scales, stream);
    else if (loads <= 192) launch_quantize_of<V, 64, 3>(x, n, dim, x_stride, codes, c_stride, scales, stream);
    else if (loads <= 256) launch_quantize_of<V, 64, 4>(x, n, dim, x_stride, codes, c_stride, scales, stream);
    else if (loads <= 384) launch_quantize_of<V, 128, 3>(x, n, dim, x_stride, codes, c_stride, scales, stream);
    else if (loads <= 512) launch_quantize_of<V, 256, 2>(x, n, dim, x_stride, codes, c_stride, scales, stream);
    else if (loads <= 768) launch_quantize_of<V, 256, 3>(x, n, dim, x_stride, codes, c_stride, scales, stream);
    else if (loads <= 1024) launch_quantize_of<V, 256, 4>(x, n, dim, x_stride, codes, c_stride, scales, stream);
    else if (loads <= 1536) launch_quantize_of<V, 256, 6>(x, n, dim, x_stride, codes, c_stride, scales, stream);
    else if (loads <= 2048) launch_quantize_of<V, 256, 8>(x, n, dim, x_stride, codes, c_stride, scales, stream);
    else hipLaunchKernelGGL((quantize_long_rows_kernel<V>), dim3((uint32_t)std::min<uint64_t>(n, 1u << 16)), dim3(1024), 0, stream, x, n, dim, x_stride, codes, c_stride, scales);
    return hipGetLastError();
}
static hipError_t launch_quantize_rows(const void* x, int value, uint64_t n, uint32_t dim, uint64_t x_stride, int8_t* codes,
                                       uint64_t c_stride, float* scales, hipStream_t stream) {
    switch (value) {
    case NEEDLE_VALUE_F32: return launch_quantize_rows_of<ValueF32>((const uint32_t*)x, n, dim, x_stride, codes, c_stride, scales, stream);
    case NEEDLE_VALUE_F16: return launch_quantize_rows_of<ValueF16>((const uint16_t*)x, n, dim, x_stride, codes, c_stride, scales, stream);
    default: return launch_quantize_rows_of<ValueBF16>((const uint16_t*)x, n, dim, x_stride, codes, c_stride, scales, stream);
    }
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
    uint32_t past;  // the output does not fit the memory-side cache and its rows start on 64 bytes: it goes past it
};

// 16 codes of a row from place `at` on, zero from k on; no word (of four bytes) without a code of the row is read.  (No 64-bit
// shifts by a lane's own amount here: with the amount in the last of a wave's 256 registers they gave wrong codes.)
template <bool ODD>
__device__ inline u32x4 load_codes(const int8_t* row, uint32_t at, uint32_t k) {
    if (at + 16 <= k) return ODD ? load16_odd(row + at) : *(const u32x4_any*)(row + at);
    if (at >= k) return u32x4{0, 0, 0, 0};
    const uint64_t first = (uint64_t)(row + at), end = (uint64_t)(row + k);
    const uint32_t by = (uint32_t)first & 3, left = k - at;  // 1 .. 15 codes
    const global_words* q = (const global_words*)(first & ~3ull);
    uint32_t w[5];
#pragma unroll
    for (uint32_t i = 0; i < 5; ++i) w[i] = (uint64_t)(q + i) < end ? q[i] : 0;
    u32x4 v;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t word = __builtin_amdgcn_alignbyte(w[i + 1], w[i], by), here = left > 4 * i ? left - 4 * i : 0;
        v[i] = here >= 4 ? word : word & ((1u << (8 * here)) - 1);
    }
    return v;
}

// Four neighbouring values of a column vector from j on; behind the last of n the last one again.
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
__device__ inline f32x4_any four_of(const float* v, uint64_t j, uint64_t n) {
    if (j + 4 <= n) return *(const f32x4_any*)(v + j);
    f32x4_any y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = v[min(j + e, n - 1)];
    return y;
}
// Four neighbouring outputs of a row from j on, as far as there are any.  Everything is in registers: a load in here would
// wait for the stores before it.
template <typename V>
__device__ inline void store_four(typename V::bits* row, uint64_t j, uint64_t n, i32x4 sums, float sa, f32x4_any sb, bool biased, f32x4_any bias) {
    typedef typename V::bits four_t __attribute__((ext_vector_type(4), aligned(V::size)));
    four_t v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float y = (float)sums[e] * sa * sb[e];
        if (biased) y += bias[e];
        v[e] = V::round(y);
    }
    if (j + 4 <= n) {
        *(four_t*)(row + j) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (j + e < n) row[j + e] = v[e];
    }
}

// ---- few rows of a ---------------------------------------------------------------------------
// At most 16 * NA rows of a: what counts is the stream over b.  A wave takes 16 * NB rows of b straight from memory into the
// matrix instruction's registers (16 bytes per lane, 64 codes of a row per load), those of a from the cache, the next slice
// under way while one is multiplied.  SPLIT: the four waves of a workgroup share the rows and take every fourth slice, so
// that a short table still has the whole chip at work; their sums meet in LDS (whole numbers: any order is exact).
template <typename V, int NB, int NA, bool SPLIT, bool ODD>
__global__ __launch_bounds__(256) void matmul_i8_stream_kernel(MatmulParams p) {
    constexpr uint32_t STEP = SPLIT ? 4 : 1;
    const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6, l15 = lane & 15, quad = lane >> 4;
    const uint64_t n0 = (SPLIT ? (uint64_t)blockIdx.x : (uint64_t)blockIdx.x * 4 + wave) * (16 * NB);
    if (!SPLIT && n0 >= p.n) return;
    const int8_t* rb[NB];
    const int8_t* ra[NA];
#pragma unroll
    for (int x = 0; x < NB; ++x) rb[x] = p.b + min(n0 + x * 16 + l15, p.n - 1) * p.b_stride + quad * 16;
#pragma unroll
    for (int y = 0; y < NA; ++y) ra[y] = p.a + (uint64_t)min(y * 16 + l15, p.m - 1) * p.a_stride + quad * 16;
    i32x4 acc[NB][NA] = {};
    u32x4 fb[2][NB], fa[2][NA];
    auto load = [&](uint32_t s, u32x4 (&b)[NB], u32x4 (&a)[NA]) {
        const uint32_t at = s * 64;
        if (at + 64 <= p.k) {
#pragma unroll
            for (int x = 0; x < NB; ++x) b[x] = ODD ? load16_odd(rb[x] + at) : *(const u32x4_any*)(rb[x] + at);
#pragma unroll
            for (int y = 0; y < NA; ++y) a[y] = ODD ? load16_odd(ra[y] + at) : *(const u32x4_any*)(ra[y] + at);
        } else {
#pragma unroll
            for (int x = 0; x < NB; ++x) b[x] = load_codes<ODD>(rb[x] - quad * 16, at + quad * 16, p.k);
#pragma unroll
            for (int y = 0; y < NA; ++y) a[y] = load_codes<ODD>(ra[y] - quad * 16, at + quad * 16, p.k);
        }
    };
    auto multiply = [&](const u32x4 (&b)[NB], const u32x4 (&a)[NA]) {
#pragma unroll
        for (int x = 0; x < NB; ++x)
#pragma unroll
            for (int y = 0; y < NA; ++y)
                acc[x][y] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, b[x]), __builtin_bit_cast(i32x4, a[y]), acc[x][y], 0, 0, 0);
    };
    const uint32_t slices = (p.k + 63) / 64;
    uint32_t s = SPLIT ? wave : 0;
    if (s < slices) load(s, fb[0], fa[0]);
    for (; s < slices; s += 2 * STEP) {
        if (s + STEP < slices) load(s + STEP, fb[1], fa[1]);
        multiply(fb[0], fa[0]);
        if (s + STEP >= slices) break;
        if (s + 2 * STEP < slices) load(s + 2 * STEP, fb[0], fa[0]);
        multiply(fb[1], fa[1]);
    }
    const uint64_t j0 = n0 + quad * 4;
    auto finish = [&](int x) {
        const uint64_t j = j0 + x * 16;
        if (j >= p.n) return;
        const f32x4_any sb = four_of(p.b_scales, j, p.n), bias = p.bias ? four_of(p.bias, j, p.n) : f32x4_any{};
#pragma unroll
        for (int y = 0; y < NA; ++y) {
            const uint32_t i = y * 16 + l15;
            if (i < p.m) store_four<V>((typename V::bits*)p.out + (uint64_t)i * p.out_stride, j, p.n, acc[x][y], p.a_scales[i], sb, p.bias != nullptr, bias);
        }
    };
    if (SPLIT) {
        __shared__ i32x4 s_part[4][NB][NA][64];
#pragma unroll
        for (int x = 0; x < NB; ++x)
#pragma unroll
            for (int y = 0; y < NA; ++y) s_part[wave][x][y][lane] = acc[x][y];
        __syncthreads();
        // wave w finishes the w-th share of the tiles of b
#pragma unroll
        for (int x = 0; x < NB; ++x) {
            if ((uint32_t)(x * 4 / NB) != wave) continue;
#pragma unroll
            for (int y = 0; y < NA; ++y) acc[x][y] = s_part[0][x][y][lane] + s_part[1][x][y][lane] + s_part[2][x][y][lane] + s_part[3][x][y][lane];
            finish(x);
        }
    } else {
#pragma unroll
        for (int x = 0; x < NB; ++x) finish(x);
    }
}

// ---- tiles through LDS -----------------------------------------------------------------------
// A workgroup of WB x WA waves makes TB rows of b x TA rows of a; a wave (TB / WB) x (TA / WA) of them with the 16x16x64
// instruction.  Slices of 64 codes pass through SLOTS LDS slots; a wave holds the operands of the slice it multiplies in
// registers and reads those of the next one meanwhile, so that slice s + 1 is read, those behind it are under way, and
// slot s, which every wave has left, takes slice s + SLOTS -- with one barrier per slice.  A slice's row is four 16-byte chunks,
// chunk c of row r at place c ^ 2 (r >> 3 & 1): the sixteen 16-byte reads that meet the banks together touch all of them
// once.  DMA: the loads write LDS themselves (rows aligned to 16 bytes, the end of a row of other than a multiple of 16 apart;
// 300 x 20000 x 777 of stride 784: 15 us, 18 through registers); otherwise they pass through registers two slices ahead,
// from any address.  SHARES: so many times the waves, each share with slots of its own and every SHARES-th slice; their sums
// meet in LDS at the end (whole numbers: any order is exact).
constexpr uint32_t SLICE = 64;
__device__ const uint32_t g_zeros[4] = {0, 0, 0, 0};
typedef __attribute__((address_space(1))) const void glb_cvoid;
typedef __attribute__((address_space(3))) void lds_void;

template <typename V, int TB, int TA, int WB, int WA, int SLOTS, bool DMA, int SHARES>
__global__ __launch_bounds__(64 * WB * WA * SHARES) void matmul_i8_tile_kernel(MatmulParams p, uint32_t tiles_b, uint32_t tiles_a) {
    constexpr int WAVES = WB * WA, NB = TB / WB / 16, NA = TA / WA / 16, STAGE = (TB + TA) * SLICE, LOADS = (TB + TA) / 16 / WAVES;
    static_assert((TB + TA) % (16 * WAVES) == 0 && TB % 16 == 0, "every wave fills whole groups of sixteen rows");
    extern __shared__ __align__(16) uint8_t s_tiles[];
    const uint32_t t = threadIdx.x, lane = t & 63, wave = (t >> 6) % WAVES, share = (t >> 6) / WAVES, l15 = lane & 15, quad = lane >> 4;
    const uint32_t wb = wave % WB, wa = wave / WB;
    uint8_t* s_tile = s_tiles + share * (SLOTS * STAGE);
    // Workgroups go to the chip's eight dies in turn, each with its own L2: a die gets a run of tiles, in groups of four
    // tiles of a that share their tiles of b.
    const uint32_t tiles = tiles_b * tiles_a;
    uint32_t tile;
    {
        const uint32_t die = blockIdx.x & 7, nth = blockIdx.x >> 3, each = tiles >> 3, more = tiles & 7;
        tile = die * each + min(die, more) + nth;
    }
    const uint32_t group = 4 * tiles_b, g0 = tile / group * 4, rows = min(4u, tiles_a - g0), in = tile % group;
    const uint32_t m0 = (g0 + in % rows) * TA;
    const uint64_t n0 = (uint64_t)(in / rows) * TB;

    // the wave's share of a slice: LOADS times sixteen rows; lane: row lane / 4, place lane % 4
    const int8_t* from[LOADS];
    const uint32_t chunk = ((lane & 3) ^ (lane >> 5 << 1)) * 16;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const uint32_t r = (wave + i * WAVES) * 16 + (lane >> 2);
        from[i] = r < TB ? p.b + min(n0 + r, p.n - 1) * p.b_stride : p.a + (uint64_t)min(m0 + r - TB, p.m - 1) * p.a_stride;
    }
    // this share's slices; how many of them the loads write themselves
    const uint32_t slices = ((p.k + SLICE - 1) / SLICE + SHARES - 1) / SHARES, full = p.k / SLICE;
    const uint32_t whole = p.k % 16 == 0 ? slices : full > share ? (full - share + SHARES - 1) / SHARES : 0;
    auto fill = [&](uint32_t s) {
        uint8_t* to = s_tile + s % SLOTS * STAGE + wave * 1024;
        const uint32_t at0 = (s * SHARES + share) * SLICE, at = at0 + chunk;
        if (at0 + SLICE <= p.k) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                __builtin_amdgcn_global_load_lds((glb_cvoid*)(from[i] + at), (lds_void*)(to + i * WAVES * 1024), 16, 0, 0);
            return;
        }
        if (p.k % 16 == 0) {  // chunks behind k are zeros
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                __builtin_amdgcn_global_load_lds((glb_cvoid*)(at < p.k ? (const void*)(from[i] + at) : (const void*)g_zeros),
                                                 (lds_void*)(to + i * WAVES * 1024), 16, 0, 0);
            return;
        }
        // the last chunk of a row in parts: through registers (`whole` does not count it)
        u32x4 end[LOADS];
#pragma unroll
        for (int i = 0; i < LOADS; ++i) end[i] = load_codes<false>(from[i], at, p.k);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) *(u32x4*)(to + lane * 16 + i * WAVES * 1024) = end[i];
    };
    auto fetch = [&](uint32_t s, u32x4 (&held)[LOADS]) {
        const uint32_t at = (s * SHARES + share) * SLICE;
        if (at + SLICE <= p.k) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) held[i] = *(const u32x4_any*)(from[i] + at + chunk);
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) held[i] = load_codes<false>(from[i], at + chunk, p.k);
        }
    };
    auto store = [&](uint32_t s, const u32x4 (&held)[LOADS]) {
        uint8_t* to = s_tile + s % SLOTS * STAGE + wave * 1024 + lane * 16;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) *(u32x4*)(to + i * WAVES * 1024) = held[i];
    };
    const uint32_t place = (quad ^ (l15 >> 3 << 1)) * 16;
    const uint32_t off_b = (wb * (TB / WB) + l15) * SLICE + place, off_a = (TB + wa * (TA / WA) + l15) * SLICE + place;
    i32x4 acc[NB][NA] = {};
    i32x4 fb[2][NB], fa[2][NA];
    auto read = [&](uint32_t s, i32x4 (&b)[NB], i32x4 (&a)[NA]) {
        const uint8_t* buf = s_tile + s % SLOTS * STAGE;
#pragma unroll
        for (int x = 0; x < NA; ++x) a[x] = *(const i32x4*)(buf + off_a + x * 16 * SLICE);
#pragma unroll
        for (int x = 0; x < NB; ++x) b[x] = *(const i32x4*)(buf + off_b + x * 16 * SLICE);
    };
    auto multiply = [&](const i32x4 (&b)[NB], const i32x4 (&a)[NA]) {
#pragma unroll
        for (int x = 0; x < NB; ++x)
#pragma unroll
            for (int y = 0; y < NA; ++y) acc[x][y] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[x], a[y], acc[x][y], 0, 0, 0);
    };
    // The reads are spread among the matrix instructions: issued in a row they would hold them up, one wave's LDS traffic
    // behind the other waves'.
    auto spread = [&] {
#pragma unroll
        for (int r = 0; r < NB + NA; ++r) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                     // an LDS read
            __builtin_amdgcn_sched_group_barrier(0x008, NB * NA / (NB + NA), 0);   // matrix instructions
        }
    };
    if (DMA) {
        // one slice: wait for slice s + 1, leave the barrier, send for slice s + SLOTS, read s + 1, multiply s
        auto step = [&](uint32_t s, int cur) {
            if (SLOTS == 4 && s + 3 < whole) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * LOADS) : "memory");
            else if (s + 2 < whole) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this wave has read slice s out of its slot
            __builtin_amdgcn_s_barrier();
            if (s + SLOTS < slices) fill(s + SLOTS);
            __builtin_amdgcn_sched_barrier(0);
            read(s + 1, fb[cur ^ 1], fa[cur ^ 1]);  // (behind the last slice: what an earlier one left there, never used)
            multiply(fb[cur], fa[cur]);
            spread();
            __builtin_amdgcn_sched_barrier(0);
        };
        for (uint32_t s = 0; s < min(slices, (uint32_t)SLOTS); ++s) fill(s);
        if (slices) {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            read(0, fb[0], fa[0]);
        }
        uint32_t s = 0;
        for (; s + 2 <= slices; s += 2) {
            step(s, 0);
            step(s + 1, 1);
        }
        if (s < slices) step(s, 0);
    } else if (slices) {
        // slot s - 1, which every wave has left, takes the slice fetched two steps ago
        u32x4 held[2][LOADS];
        auto step = [&](uint32_t s, int cur) {
            __syncthreads();
            if (s + SLOTS - 1 < slices) store(s + SLOTS - 1, held[(cur + SLOTS - 1) & 1]);
            if (s + SLOTS + 1 < slices) fetch(s + SLOTS + 1, held[(cur + SLOTS - 1) & 1]);
            __builtin_amdgcn_sched_barrier(0);
            read(s + 1, fb[cur ^ 1], fa[cur ^ 1]);
            multiply(fb[cur], fa[cur]);
            spread();
            __builtin_amdgcn_sched_barrier(0);
        };
        for (uint32_t s = 0; s < min(slices, SLOTS - 1u); ++s) {
            fetch(s, held[0]);
            store(s, held[0]);
        }
        if (SLOTS - 1 < slices) fetch(SLOTS - 1, held[(SLOTS - 1) & 1]);
        if (SLOTS < slices) fetch(SLOTS, held[SLOTS & 1]);
        __syncthreads();
        read(0, fb[0], fa[0]);
        uint32_t s = 0;
        for (; s + 2 <= slices; s += 2) {
            step(s, 0);
            step(s + 1, 1);
        }
        if (s < slices) step(s, 0);
    }
    if (SHARES > 1) {  // the sums of the other shares meet in LDS
        i32x4* sums = (i32x4*)s_tiles + (wave * 64 + lane);
        constexpr uint32_t STEP = WAVES * 64;
        __syncthreads();
        if (share) {
#pragma unroll
            for (int x = 0; x < NB; ++x)
#pragma unroll
                for (int y = 0; y < NA; ++y) sums[((share - 1) * NB * NA + x * NA + y) * STEP] = acc[x][y];
        }
        __syncthreads();
        if (!share) {
#pragma unroll
            for (int o = 0; o < SHARES - 1; ++o)
#pragma unroll
                for (int x = 0; x < NB; ++x)
#pragma unroll
                    for (int y = 0; y < NA; ++y) acc[x][y] += sums[(o * NB * NA + x * NA + y) * STEP];
        }
    }
    const uint64_t j0 = n0 + wb * (TB / WB) + quad * 4;
    const uint32_t i0 = m0 + wa * (TA / WA) + l15;
    f32x4_any sb[NB], bias[NB];
    float sa[NA];
#pragma unroll
    for (int x = 0; x < NB; ++x) {
        sb[x] = four_of(p.b_scales, j0 + x * 16, p.n);
        bias[x] = p.bias ? four_of(p.bias, j0 + x * 16, p.n) : f32x4_any{-0.0f, -0.0f, -0.0f, -0.0f};  // x + -0 is x
    }
#pragma unroll
    for (int y = 0; y < NA; ++y) sa[y] = p.a_scales[min(i0 + y * 16, p.m - 1)];
    typedef typename V::bits four_t __attribute__((ext_vector_type(4), aligned(V::size)));
    auto four = [&](int x, int y) {
        four_t v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = V::round((float)acc[x][y][e] * sa[y] * sb[x][e] + bias[x][e]);
        return v;
    };
    typename V::bits* o = (typename V::bits*)p.out + (uint64_t)i0 * p.out_stride + j0;
    if (n0 + TB <= p.n && m0 + TA <= p.m) {
        // Through the wave's own part of LDS, so that a store writes whole lines: 16 bytes per lane along a row instead of
        // four outputs here and there.  16-byte chunk c of row r lies at place c ^ r (mod the row's chunks).
        constexpr int LINE = TB / WB * V::size, CHUNKS = LINE / 16, GO = 64 / CHUNKS;  // bytes and chunks of a row; rows per store
        constexpr int PASS = V::size == 4 ? 1 : NA, ROWS = PASS * 16;  // f32: sixteen rows at a time
        static_assert(ROWS * LINE * WAVES <= SLOTS * STAGE && CHUNKS <= 64 && ROWS % GO == 0, "the waves' parts fit");
        uint8_t* part = s_tile + wave * (ROWS * LINE);
        __syncthreads();
        if (share) return;
        o = (typename V::bits*)p.out + (uint64_t)(m0 + wa * (TA / WA)) * p.out_stride + n0 + wb * (TB / WB);
#pragma unroll
        for (int y0 = 0; y0 < NA; y0 += PASS) {
#pragma unroll
            for (int y = 0; y < PASS; ++y)
#pragma unroll
                for (int x = 0; x < NB; ++x) {
                    const uint32_t r = y * 16 + l15, byte = (x * 16 + quad * 4) * V::size;
                    *(four_t*)__builtin_assume_aligned(part + r * LINE + (((byte >> 4) ^ r) & (CHUNKS - 1)) * 16 + (byte & 15), 4 * V::size) = four(x, y0 + y);
                }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int g = 0; g < ROWS / GO; ++g) {
                const uint32_t r = g * GO + lane / CHUNKS, c = lane % CHUNKS;
                const u32x4 v = *(const u32x4*)(part + r * LINE + ((c ^ r) & (CHUNKS - 1)) * 16);
                u32x4_any* to = (u32x4_any*)((uint8_t*)(o + (uint64_t)(y0 * 16 + r) * p.out_stride) + c * 16);
                if (p.past) {
                    asm volatile("");  // (without these the compiler makes one ordinary store of the two)
                    __builtin_nontemporal_store(v, to);
                    asm volatile("");
                } else {
                    *to = v;
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
    } else if (!share) {
#pragma unroll
        for (int y = 0; y < NA; ++y) {
            if (i0 + y * 16 >= p.m) continue;
#pragma unroll
            for (int x = 0; x < NB; ++x) {
                const four_t v = four(x, y);
                typename V::bits* at = o + (uint64_t)(y * 16) * p.out_stride + x * 16;
                if (j0 + x * 16 + 4 <= p.n) {
                    *(four_t*)at = v;
                } else {
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        if (j0 + x * 16 + e < p.n) at[e] = v[e];
                }
            }
        }
    }
}

template <typename V, int TB, int TA, int WB, int WA, int SLOTS, bool DMA, int SHARES = 1>
static hipError_t launch_tiles_of(const MatmulParams& p, hipStream_t stream) {
    constexpr uint32_t lds = SHARES * SLOTS * (TB + TA) * SLICE;
    if (lds >= 65536) {  // (per device, like every attribute of a kernel)
        const hipError_t e =
            hipFuncSetAttribute((const void*)matmul_i8_tile_kernel<V, TB, TA, WB, WA, SLOTS, DMA, SHARES>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    const uint32_t tiles_b = (uint32_t)((p.n + TB - 1) / TB), tiles_a = (p.m + TA - 1) / TA;
    hipLaunchKernelGGL((matmul_i8_tile_kernel<V, TB, TA, WB, WA, SLOTS, DMA, SHARES>), dim3(tiles_b * tiles_a), dim3(64 * WB * WA * SHARES), lds, stream, p, tiles_b, tiles_a);
    return hipGetLastError();
}
// From this k on the few tiles of a small product share it among four times the waves: 512 x 512 x 4096 takes 13 us so, 18
// without; 64 x 1000 x 4096 9 and 14; 500 x 700 x 768 5 either way, 1000 x 1000 x 1024 7.5 and 6.6.
constexpr uint32_t SHARED_K = 2048;
constexpr uint64_t ALIGN_MOST = 2ull << 30;  // workspace of the aligned copies; beyond it the rows pass through registers
// The rows of b and of a copied to rows of `to_stride` (a multiple of 64) with zeros behind them, a wave per row.
__global__ __launch_bounds__(256) void align_rows_kernel(MatmulParams p, int8_t* __restrict__ to, uint32_t to_stride) {
    const uint64_t row = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= p.n + p.m) return;
    const int8_t* from = row < p.n ? p.b + row * p.b_stride : p.a + (row - p.n) * p.a_stride;
    for (uint32_t at = (threadIdx.x & 63) * 16; at < to_stride; at += 1024) *(u32x4*)(to + row * to_stride + at) = load_codes<true>(from, at, p.k);
}

// Rows that do not all start on a multiple of four: the kernel for few rows loads them by words.  The tiles hide what such
// loads cost behind their sums (112 x 14225 x 1971: 17 us, 20 by words).
static bool rows_odd(const MatmulParams& p) {
    return (((uintptr_t)p.a | (uintptr_t)p.b | (p.m > 1 ? p.a_stride : 0) | (p.n > 1 ? p.b_stride : 0)) & 3) != 0;
}
template <typename V, int NB, int NA, bool SPLIT>
static hipError_t launch_stream_of(const MatmulParams& p, hipStream_t stream) {
    const uint64_t tiles = (p.n + 16 * NB - 1) / (16 * NB);
    const dim3 grid((uint32_t)(SPLIT ? tiles : (tiles + 3) / 4));
    if (rows_odd(p)) hipLaunchKernelGGL((matmul_i8_stream_kernel<V, NB, NA, SPLIT, true>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((matmul_i8_stream_kernel<V, NB, NA, SPLIT, false>), grid, dim3(256), 0, stream, p);
    return hipGetLastError();
}
static bool rows_aligned(const MatmulParams& p) {
    return p.a_stride % 16 == 0 && p.b_stride % 16 == 0 && (uintptr_t)p.a % 16 == 0 && (uintptr_t)p.b % 16 == 0;
}
static uint64_t tiles_of(const MatmulParams& p, uint64_t tb, uint64_t ta) { return ((p.n + tb - 1) / tb) * ((p.m + ta - 1) / ta); }

template <typename V>
static hipError_t launch_matmul_of(const MatmulParams& p, int n_cu, hipStream_t stream) {
    const bool aligned = rows_aligned(p);
    if (p.m <= 16) {
        // split: long rows of a short table.  Otherwise many short-lived waves of one tile each hide the latency best.
        const bool split = p.n < 256ull * n_cu && p.k > 256;
        if (!split) return launch_stream_of<V, 1, 1, false>(p, stream);
        return p.n < 64ull * n_cu ? launch_stream_of<V, 2, 1, true>(p, stream) : launch_stream_of<V, 4, 1, true>(p, stream);
    }
    // Tiles, by what fills the chip (us of the kernel, sizes m x n x k).  A long product of many 256 x 256 tiles is bound by the
    // matrix cores and the power they draw: 8192 x 8192 x 4096 takes 247 with them, 480 with 128 x 128.  One such tile per CU
    // takes about (2.8 + 512 / k) times one of 128 x 128 per CU, and what counts is how often the chip is filled: 4096 x
    // 4096 x 2048 (1 and 4 fills) 32 with 256 x 256, 38 with 128 x 128; 4096 x 4352 x 2048 (2 and 5) 57 and 46; 4096 x 6144 x
    // 4096 (2 and 6) 106 and 115; 2048 x 2048 x 2048 38 and 21.  Short ones: 1000 x 100000 x 128, bound by its output, 110 and
    // 98.  Below half a tile per CU 128 x 64 and 64 x 64 (512 x 512 x 4096: 18 with 64 x 64 and one share, 25 with 128 x 128).  Through
    // registers 256 x 128 are the largest, and taken where they come to two per CU.
    const auto tiles = [&](uint64_t tb, uint64_t ta) { return tiles_of(p, tb, ta); };
    const uint64_t cu = (uint64_t)n_cu;
    const auto fills = [&](uint64_t of) { return (of + cu - 1) / cu; };
    if (p.m > 128 && p.k >= 512) {
        if (aligned && (28 + 5120 / p.k) * fills(tiles(256, 256)) < 10 * fills(tiles(128, 128))) return launch_tiles_of<V, 256, 256, 2, 4, 4, true>(p, stream);
        if (!aligned && tiles(256, 256) >= cu) return launch_tiles_of<V, 256, 128, 4, 2, 4, false>(p, stream);
    }
    if (p.m > 64 && tiles(128, 128) >= cu / 2)
        return aligned ? launch_tiles_of<V, 128, 128, 4, 2, 4, true>(p, stream) : launch_tiles_of<V, 128, 128, 4, 2, 4, false>(p, stream);
    if (tiles(128, 64) >= cu)
        return aligned ? launch_tiles_of<V, 128, 64, 2, 2, 4, true>(p, stream) : launch_tiles_of<V, 128, 64, 2, 2, 4, false>(p, stream);
    if (p.k >= SHARED_K && tiles(64, 64) <= cu)
        return aligned ? launch_tiles_of<V, 64, 64, 2, 2, 4, true, 4>(p, stream) : launch_tiles_of<V, 64, 64, 2, 2, 4, false, 4>(p, stream);
    return aligned ? launch_tiles_of<V, 64, 64, 2, 2, 4, true>(p, stream) : launch_tiles_of<V, 64, 64, 2, 2, 4, false>(p, stream);
}
static hipError_t launch_slab(needle_hip_ctx* c, MatmulParams p, int out_value) {
    // 1000 x 100000 x 128 to 400 MB of f32: 81 us past the cache, 103 through it; to 134 MB of bf16 (8192 x 8192 x 64) 37 and
    // 32; where rows do not start on 64 bytes (1000 x 100003) 190 and 106.
    const uint64_t size = value_size(out_value);
    p.past = p.m * p.n * size > (256ull << 20) && (uintptr_t)p.out % 64 == 0 && p.out_stride * size % 64 == 0;
    // Rows that the loads cannot write to LDS themselves (odd k, strides or addresses): a product of more tiles than CUs copies
    // them to rows that can be first, where enough sums are made of each code.  us of the copies and the product, and of the
    // product through registers: 8192 x 8192 x 1000 104, 145; 2256 x 6573 x 1946 62, 83; 4196 x 5755 x 218 28, 34; 600 x 60000 x
    // 513 62, 64; not so 300 x 66000 x 513 63, 46; 2000 x 2000 x 301 11, 7.
    const uint32_t stride = (p.k + 63) / 64 * 64;
    const uint64_t bytes = (p.n + p.m) * stride;
    bool copy = !rows_aligned(p) && tiles_of(p, 128, 128) > (uint64_t)c->n_cu && p.m * p.n >= 512 * (p.m + p.n) && bytes <= ALIGN_MOST;
    if (copy) {
        const hipError_t e = c->scratch[5].ensure(bytes);
        if (e == hipErrorOutOfMemory) {  // the product needs no copies: on as the rows are
            (void)hipGetLastError();
            copy = false;
        } else if (e != hipSuccess) {
            return e;
        }
    }
    if (copy) {
        int8_t* to = c->scratch[5].as<int8_t>();
        hipLaunchKernelGGL(align_rows_kernel, dim3((uint32_t)((p.n + p.m + 3) / 4)), dim3(256), 0, c->stream, p, to, stride);
        p.b = to;
        p.a = to + p.n * stride;
        p.a_stride = p.b_stride = p.k = stride;
    }
    switch (out_value) {
    case NEEDLE_VALUE_F32: return launch_matmul_of<ValueF32>(p, c->n_cu, c->stream);
    case NEEDLE_VALUE_F16: return launch_matmul_of<ValueF16>(p, c->n_cu, c->stream);
    default: return launch_matmul_of<ValueBF16>(p, c->n_cu, c->stream);
    }
}

// Slabs of rows whose grids stay below 2^32 threads, the most a launch takes: the largest have a workgroup of 512 for every
// tile of 128 x 128 (smaller tiles are taken for products of few).
constexpr uint64_t SLAB_N = 1ull << 26, SLAB_M = 1ull << 22, SLAB_TILES = 1ull << 22;
constexpr uint64_t slab_rows(uint64_t n) {  // of a, against n <= SLAB_N rows of b
    const uint64_t rows = SLAB_TILES / ((n + 127) / 128) * 128;
    return rows < SLAB_M ? rows : SLAB_M;
}
static_assert(slab_rows(SLAB_N) >= 128 && (slab_rows(SLAB_N) / 128) * (SLAB_N / 128) * 512 < (1ull << 32) &&
              (slab_rows((1u << 22) + 1) / 128) * ((1u << 15) + 1) * 512 < (1ull << 32), "a launch takes the grid");
static hipError_t launch_matmul_i8(needle_hip_ctx* c, const MatmulParams& p, int out_value) {
    const uint64_t most = slab_rows(std::min(SLAB_N, p.n));
    for (uint64_t i = 0; i < p.m; i += most)
        for (uint64_t j = 0; j < p.n; j += SLAB_N) {
            MatmulParams q = p;
            q.m = (uint32_t)std::min(most, p.m - i);
            q.n = std::min(SLAB_N, p.n - j);
            q.a += i * p.a_stride;
            q.a_scales += i;
            q.b += j * p.b_stride;
            q.b_scales += j;
            if (p.bias) q.bias += j;
            q.out = (unsigned char*)p.out + (i * p.out_stride + j) * value_size(out_value);
            const hipError_t e = launch_slab(c, q, out_value);
            if (e != hipSuccess) return e;
        }
    return hipSuccess;
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
    if (n >= (1ull << 31) || m >= (1u << 31)) return fail(NEEDLE_HIP_ERR_UNSUPPORTED, "at most 2^31-1 rows of a and of b");
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
    HIP_TRY(wait_done(c));
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
    const MatmulParams p{d_a, d_b, d_a_scales, d_b_scales, d_bias, d_out, a_stride, b_stride, out_stride, n, m, k, 0};
    HIP_TRY(launch_matmul_i8(c, p, out_value));
    HIP_TRY(wait_done(c));
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
                         bias ? (const float*)(d + at[4]) : nullptr, d + at[5], k, k, n, n, m, k, 0};
    HIP_TRY(launch_matmul_i8(c, p, NEEDLE_VALUE_F32));
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
    const MatmulParams p{d_codes, d_b, d_scales, d_b_scales, d_bias, d_out, stride, b_stride, out_stride, n, m, k, 0};
    HIP_TRY(launch_matmul_i8(c, p, out_value));
    HIP_TRY(wait_done(c));
    return NEEDLE_HIP_OK;
}
