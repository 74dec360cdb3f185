// lmr_rows.hpp — the row operators' arguments and element types (lmr_rows.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>
#include "../../include/lamellar_gpu_ops.h"

namespace lmr {

struct RowTable {
    void* data;          // rows x row_len elements
    float* scales;       // 8-bit types: rows x groups
    uint32_t* claims;    // rows words, zero between calls (null: the caller's rows are distinct)
    uint64_t rows;
    uint32_t row_len, type;
    uint32_t group, groups;   // elements of a group, groups of a row (other types: the whole row, 1)
};
struct RowBatch {
    const void* idx;
    uint32_t index_size;
    bool has_pad;
    int64_t pad;
    uint64_t n;
    float scale;
    uint64_t stride;     // elements between two records' values
};

struct code_i8 { int8_t b; };
struct code_e4m3 { uint8_t b; };
template <typename T> struct is_code { static constexpr bool v = false; };
template <> struct is_code<code_i8> { static constexpr bool v = true; };
template <> struct is_code<code_e4m3> { static constexpr bool v = true; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return float(v); }
__device__ __forceinline__ float to_f32(__bf16 v) { return float(v); }
__device__ __forceinline__ float to_f32(code_i8 v) { return float(v.b); }
__device__ __forceinline__ float to_f32(code_e4m3 v) { return __builtin_amdgcn_cvt_f32_fp8(int(v.b), 0); }

template <typename T> __device__ __forceinline__ T from_f32(float v) { return T(v); }

// Eight elements of a row at a time, from and to addresses aligned to one element (a row of odd
// length starts anywhere): the device's vector loads take any address, so no aligned form is needed.
constexpr int kChunk = 8;
template <typename T> struct Chunk { uint32_t w[kChunk * sizeof(T) / 4]; };

template <typename T>
__device__ __forceinline__ Chunk<T> load_chunk(const T* p) {
    Chunk<T> c;
    __builtin_memcpy(&c, p, sizeof(c));
    return c;
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* p, const Chunk<T>& c) {
    __builtin_memcpy(p, &c, sizeof(c));
}
// the same for data that the caches need not keep
template <typename T>
__device__ __forceinline__ void stream_chunk(T* p, const Chunk<T>& c) {
    typedef uint32_t x4 __attribute__((ext_vector_type(4), aligned(2)));
    x4 v[sizeof(c) / 16];
    __builtin_memcpy(v, &c, sizeof(c));
#pragma unroll
    for (unsigned i = 0; i < sizeof(c) / 16; i++) __builtin_nontemporal_store(v[i], reinterpret_cast<x4*>(p) + i);
}
// The last chunk of a row whose length is no multiple of 8 is the row's last 8 elements: it overlaps
// the one before, and [lo, hi) are the elements it has for itself. So every access is one whole vector.
// A chunk behind the row's end has none. Rows shorter than 8 are one chunk, read element by element.
struct Span { uint32_t at; int lo, hi; };
__device__ __forceinline__ Span span_of(uint32_t chunk, uint32_t len) {
    const uint32_t col = chunk * kChunk;
    if (len < kChunk) return {0, 0, chunk == 0 ? int(len) : 0};
    if (col + kChunk <= len) return {col, 0, kChunk};
    return {len - kChunk, col < len ? kChunk - int(len - col) : kChunk, kChunk};
}
// (zeros where `on` is false; LONG: the caller knows that rows have at least 8 elements)
template <bool LONG = false, typename T>
__device__ __forceinline__ Chunk<T> fetch(const T* p, uint32_t at, uint32_t len, bool on) {
    Chunk<T> c = {};
    if (LONG || len >= kChunk) {
        if (on) c = load_chunk(p + at);
    } else if (on) {
        T e[kChunk] = {};
#pragma unroll
        for (int i = 0; i < kChunk; i++) if (i < int(len)) e[i] = p[i];
        __builtin_memcpy(&c, e, sizeof(c));
    }
    return c;
}
template <typename T>
__device__ __forceinline__ void put_some(T* p, const Chunk<T>& c, int lo, int hi) {
    T e[kChunk];
    __builtin_memcpy(e, &c, sizeof(c));
#pragma unroll
    for (int i = 0; i < kChunk; i++) if (i >= lo && i < hi) p[i] = e[i];
}
// the whole chunk, where two that overlap write the same values
template <typename T>
__device__ __forceinline__ void put(T* p, uint32_t at, uint32_t len, const Chunk<T>& c) {
    if (len >= kChunk) store_chunk(p + at, c);
    else put_some(p, c, 0, int(len));
}
// its own elements only
template <typename T>
__device__ __forceinline__ void put_own(T* p, const Span& s, const Chunk<T>& c) {
    if (s.lo == 0 && s.hi == kChunk) store_chunk(p + s.at, c);
    else put_some(p + s.at, c, s.lo, s.hi);
}
template <typename T>
__device__ __forceinline__ void unpack(const Chunk<T>& c, float (&v)[kChunk]) {
    if constexpr (std::is_same_v<T, __bf16>) {
#pragma unroll
        for (int i = 0; i < kChunk; i++) v[i] = __uint_as_float(i & 1 ? c.w[i / 2] & 0xffff0000u : c.w[i / 2] << 16);
    } else if constexpr (std::is_same_v<T, code_e4m3>) {
#pragma unroll
        for (int i = 0; i < kChunk; i += 2) {
            const auto f = i & 2 ? __builtin_amdgcn_cvt_pk_f32_fp8(int(c.w[i / 4]), true)
                                 : __builtin_amdgcn_cvt_pk_f32_fp8(int(c.w[i / 4]), false);
            v[i] = f[0];
            v[i + 1] = f[1];
        }
    } else {
        T e[kChunk];
        __builtin_memcpy(e, &c, sizeof(c));
#pragma unroll
        for (int i = 0; i < kChunk; i++) v[i] = to_f32(e[i]);
    }
}
template <typename T>
__device__ __forceinline__ Chunk<T> pack(const float (&v)[kChunk]) {
    T e[kChunk];
#pragma unroll
    for (int i = 0; i < kChunk; i++) e[i] = from_f32<T>(v[i]);
    Chunk<T> c;
    __builtin_memcpy(&c, e, sizeof(c));
    return c;
}

// x / d by multiplication with 2^64 / d (2^32 / d) rounded up: exact while x * d stays below 2^64 (2^32).
// Here d is at most 2^15 (the chunks of the longest row) and x below 2^34, 2^16 where it has 32 bits.
struct Divisor { uint32_t d, m32; uint64_t m64; };
inline Divisor divisor(uint32_t d) {
    return {d, d > 1 ? uint32_t((uint64_t(1) << 32) / d + 1) : 0u, d > 1 ? ~uint64_t(0) / d + 1 : 0u};
}
__device__ __forceinline__ uint64_t quotient64(uint64_t x, const Divisor& d) { return d.d > 1 ? __umul64hi(x, d.m64) : x; }
__device__ __forceinline__ uint32_t quotient32(uint32_t x, const Divisor& d) { return d.d > 1 ? __umulhi(x, d.m32) : x; }

// A group's scale from its largest |x| (as bits). The floor keeps 1 / scale finite; an infinity or
// NaN in the group makes the scale NaN, and the codes 0, so that the whole group reads back as NaN:
// 8-bit integers have no code for it, and a finite scale would hide it.
struct GroupScale { float scale, inv; };
template <typename T>
__device__ __forceinline__ GroupScale group_scale(uint32_t max_bits) {
    constexpr float inv_q = is_code<T>::v && std::is_same_v<T, code_i8> ? float(1.0 / 127.0) : float(1.0 / 448.0);
    if (max_bits >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.f};
    const float s = fmaxf(__uint_as_float(max_bits) * inv_q, 1.17549435e-38f);
    return {s, 1.0f / s};
}
}  // namespace lmr
