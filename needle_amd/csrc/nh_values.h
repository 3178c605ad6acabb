// Arrays in floating point that an operator takes or gives in one of three types (needle_value), and what the host side
// of such operators checks.
#pragma once
#include "nh_api.h"

namespace nh {

__host__ __device__ inline uint32_t value_size(int value) { return value == NEEDLE_VALUE_F32 ? 4u : 2u; }
inline bool value_known(int value) {
    return value == NEEDLE_VALUE_F32 || value == NEEDLE_VALUE_F16 || value == NEEDLE_VALUE_BF16;
}

// A loaded pattern widened to f32 (exact), and an f32 rounded to the type (nearest, ties to even).
struct ValueF32 {
    typedef uint32_t bits;
    static constexpr int size = 4;
    __device__ static float widen(uint32_t u) { return __uint_as_float(u); }
    __device__ static uint32_t round(float f) { return __float_as_uint(f); }
};
struct ValueF16 {
    typedef uint16_t bits;
    static constexpr int size = 2;
    __device__ static float widen(uint16_t u) { return (float)__builtin_bit_cast(_Float16, u); }
    __device__ static uint16_t round(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
};
struct ValueBF16 {
    typedef uint16_t bits;
    static constexpr int size = 2;
    __device__ static float widen(uint16_t u) { return __uint_as_float((uint32_t)u << 16); }
    __device__ static uint16_t round(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
};

// 16 bytes at any address: the target's global loads and stores need no alignment.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(1)));

// The same 16 bytes where the address need not even be a multiple of four.  A load from such an address is taken apart by the
// memory pipeline (1 x 9856 x 3569 codes of odd stride: 32 us with it, 19 with this): so the whole words that hold the bytes are
// read and shifted into place.  No word without one of the bytes is read.
typedef __attribute__((address_space(1))) uint32_t global_words;
typedef u32x4 u32x4_words __attribute__((aligned(4)));
typedef __attribute__((address_space(1))) u32x4_words global_words4;
__device__ inline u32x4 load16_odd(const void* p) {
    const uint32_t by = (uint32_t)(uint64_t)p & 3;
    const global_words* q = (const global_words*)((uint64_t)p & ~3ull);
    const u32x4 v = *(const global_words4*)q;
    const uint32_t w = q[by ? 4 : 3];
    return u32x4{__builtin_amdgcn_alignbyte(v[1], v[0], by), __builtin_amdgcn_alignbyte(v[2], v[1], by),
                 __builtin_amdgcn_alignbyte(v[3], v[2], by), __builtin_amdgcn_alignbyte(w, v[3], by)};
}

// Makes `device` current for one call and gives the caller's own back on return.
class DeviceScope {
public:
    explicit DeviceScope(int device) {
        e_ = hipGetDevice(&was_);
        if (e_ == hipSuccess && was_ != device) {
            e_ = hipSetDevice(device);
            moved_ = e_ == hipSuccess;
        }
    }
    ~DeviceScope() {
        if (moved_) (void)hipSetDevice(was_);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
    hipError_t error() const { return e_; }
private:
    int was_ = 0;
    bool moved_ = false;
    hipError_t e_ = hipSuccess;
};

// Bytes from the first to behind the last element of `rows` rows of `len` elements, `stride` apart; false on overflow.
inline bool span_bytes(uint64_t rows, uint64_t len, uint64_t stride, uint64_t size, uint64_t* out) {
    *out = 0;
    if (rows == 0 || len == 0) return true;
    uint64_t last, all;
    if (__builtin_mul_overflow(rows - 1, stride, &last) || __builtin_add_overflow(last, len, &all) ||
        __builtin_mul_overflow(all, size, &all) || all > (1ull << 62))
        return false;
    *out = all;
    return true;
}
inline bool ranges_meet(const void* a, uint64_t na, const void* b, uint64_t nb) {
    const uint64_t x = (uint64_t)a, y = (uint64_t)b;
    return a && b && na && nb && x < y + nb && y < x + na;
}

// Waits until everything on the context's stream has finished; the caller holds the context's lock.
hipError_t wait_done(needle_hip_ctx* c);

}  // namespace nh
