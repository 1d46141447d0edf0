// Shared device-side definitions of the 8-bit paged cache (include/ffnrm.h, ffnrm_kv_*).
//
// Pools: codes int8 [layers][pages][kv_heads][page_tokens][head_dim], scales f32
// [layers][pages][kv_heads], one pair for K and one for V; value = code * scale. A step is a
// batch of sequences: tables [seqs][width] of page ids, lengths [seqs] (tokens held with the
// step's new ones) and starts [seqs + 1], the rows of the new tokens. New token j of a
// sequence's n stands at position length - n + j; a sequence of length 0 is idle.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace ffnrm::kv {

// Bits of the handle's status word, set by kernels that met data they cannot use.
constexpr int kStatusPage = 1;      // a page id outside the pool
constexpr int kStatusLength = 2;    // a length or row count that does not fit the tables or the rows
constexpr int kStatusRotary = 4;    // a position past the end of the rotary table
constexpr int kStatusPages = 8;     // not enough free pages
constexpr int kStatusWait = 16;     // a bounded pipeline wait ran out

// One layer's pools and the geometry.
struct Pool {
    int8_t *k_codes, *v_codes;
    float *k_scale, *v_scale;
    int pages, heads, dim, page_tokens, page_shift;
};

// One step's batch. starts == nullptr: one row per sequence.
struct Batch {
    const int32_t *tables, *lengths, *starts;
    int seqs, width, rows;
};

// Row range of a sequence; a range outside [0, rows] is reported and taken as empty.
__device__ __forceinline__ bool seq_rows(const Batch &b, int s, int &first, int &count) {
    first = s;
    count = 1;
    if (b.starts) {
        first = b.starts[s];
        count = b.starts[s + 1] - first;
    }
    if (first < 0 || count < 0 || first > b.rows || count > b.rows - first) {
        first = count = 0;
        return false;
    }
    return true;
}

// A sequence's token count, held to what its table row can address.
__device__ __forceinline__ bool seq_length(const Batch &b, int s, int page_shift, int &length) {
    length = b.lengths[s];
    if (length < 0 || length > (int64_t(b.width) << page_shift)) {
        length = 0;
        return false;
    }
    return true;
}

// The sequence that row r belongs to: the last s with starts[s] <= r (32 probes per round,
// whole warp). starts are non-decreasing; any other content gives some s in [0, seqs).
__device__ __forceinline__ int seq_of_row(const int32_t *starts, int seqs, int r) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = seqs;  // answer in [lo, hi)
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int probe = lo + lane * step;
        const unsigned m = __ballot_sync(0xffffffffu, probe < hi && starts[probe] <= r);
        const int last = m ? 31 - __clz(m) : 0;
        lo += last * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

// A stored scale as the kernels take it: finite and not negative, else NaN.
__device__ __forceinline__ float sound_scale(float s) {
    return s >= 0.f && s < __int_as_float(0x7f800000) ? s : __int_as_float(0x7fffffff);
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }

// N elements in one aligned access (N * sizeof(T) is 16 or 32 bytes).
template <typename T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Vec {
    T v[N];
};

// N values to and from f32, two to an instruction where the type allows.
template <typename T, int N>
__device__ __forceinline__ void unpack(const Vec<T, N> &v, float *f) {
    if constexpr (N % 2 == 0 && sizeof(T) == 2) {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const T2 p = *reinterpret_cast<const T2 *>(&v.v[i]);
            float2 x;
            if constexpr (std::is_same<T, __half>::value)
                x = __half22float2(p);
            else
                x = __bfloat1622float2(p);
            f[i] = x.x, f[i + 1] = x.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = to_f32(v.v[i]);
    }
}
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> pack(const float *f) {
    Vec<T, N> v;
    if constexpr (N % 2 == 0 && sizeof(T) == 2) {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            T2 p;
            if constexpr (std::is_same<T, __half>::value)
                p = __floats2half2_rn(f[i], f[i + 1]);
            else
                p = __floats2bfloat162_rn(f[i], f[i + 1]);
            *reinterpret_cast<T2 *>(&v.v[i]) = p;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v.v[i] = from_f32<T>(f[i]);
    }
    return v;
}

// The rotation of one pair in f32, every product and sum rounded by itself so that the
// result does not depend on contraction: (a c - b s, b c + a s).
__device__ __forceinline__ void rotate_pair(float &a, float &b, float c, float s) {
    const float y = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
    a = y;
}

}  // namespace ffnrm::kv
