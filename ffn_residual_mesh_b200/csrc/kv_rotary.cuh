// Rotary positions. For a head row x and R rotated channels, pair i < R/2 is
// (x[i], x[i + R/2]) (half layout) or (x[2i], x[2i + 1]) (interleaved) and becomes
// (a c - b s, b c + a s) with c, s = row `position` of the cos | sin table; channels R.. are
// copied. The inverse takes -s: the transposed rotation, which is also the gradient. f32
// arithmetic, one rounding to the output type.
#pragma once

#include "kv_common.cuh"

namespace ffnrm::kv {

struct RotaryArgs {
    const void *x;
    void *y;
    const int32_t *positions;
    const float *table;  // [max_positions][R]: R/2 cosines, then R/2 sines
    int64_t x_token, x_head, y_token, y_head;  // strides in elements
    int tokens, heads, dim, rot, max_positions;
};

// Units of one head row: with VEC channels per access, a unit is a pair of VEC-channel
// runs (half layout), VEC channels (interleaved), or VEC copied channels. VEC = 1 takes
// one pair or one copied channel.
template <bool INTERLEAVED, int VEC>
__host__ __device__ constexpr int rotary_units(int dim, int rot) {
    return ((INTERLEAVED && VEC > 1) ? rot : rot / 2) / VEC + (dim - rot) / VEC;
}

// Whether VEC channels at a time cover the row's halves and rest.
template <bool INTERLEAVED, int VEC>
constexpr bool rotary_fits(int dim, int rot) {
    return dim % VEC == 0 && rot % VEC == 0 && (INTERLEAVED || (rot / 2) % VEC == 0);
}

// Rotates unit u of the head row x into y (which may be x). `table` is the position's row,
// nullptr for a position outside the table: the rotated channels become NaN.
template <typename T, bool INTERLEAVED, int VEC>
__device__ __forceinline__ void rotate_unit(const T *x, T *y, const float *table, int u, int dim, int rot, float sign) {
    const int half = rot / 2;
    const int rotated = ((INTERLEAVED && VEC > 1) ? rot : half) / VEC;
    if (u >= rotated) {
        const int d = rot + (u - rotated) * VEC;
        *reinterpret_cast<Vec<T, VEC> *>(y + d) = *reinterpret_cast<const Vec<T, VEC> *>(x + d);
        return;
    }
    const float nan = __int_as_float(0x7fffffff);
    if constexpr (INTERLEAVED && VEC > 1) {
        Vec<T, VEC> v = *reinterpret_cast<const Vec<T, VEC> *>(x + u * VEC);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            const int p = u * (VEC / 2) + i;
            float a = to_f32(v.v[2 * i]), b = to_f32(v.v[2 * i + 1]);
            rotate_pair(a, b, table ? table[p] : nan, table ? sign * table[half + p] : nan);
            v.v[2 * i] = from_f32<T>(a);
            v.v[2 * i + 1] = from_f32<T>(b);
        }
        *reinterpret_cast<Vec<T, VEC> *>(y + u * VEC) = v;
    } else {
        const int ia = INTERLEAVED ? 2 * u : u * VEC, ib = INTERLEAVED ? 2 * u + 1 : u * VEC + half;
        Vec<T, VEC> va = *reinterpret_cast<const Vec<T, VEC> *>(x + ia), vb = *reinterpret_cast<const Vec<T, VEC> *>(x + ib);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int p = u * VEC + i;
            float a = to_f32(va.v[i]), b = to_f32(vb.v[i]);
            rotate_pair(a, b, table ? table[p] : nan, table ? sign * table[half + p] : nan);
            va.v[i] = from_f32<T>(a);
            vb.v[i] = from_f32<T>(b);
        }
        *reinterpret_cast<Vec<T, VEC> *>(y + ia) = va;
        *reinterpret_cast<Vec<T, VEC> *>(y + ib) = vb;
    }
}

// One thread per unit of one head row.
template <typename T, bool INTERLEAVED, int VEC>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs a, float sign) {
    const int units = rotary_units<INTERLEAVED, VEC>(a.dim, a.rot);
    const int64_t n = int64_t(a.tokens) * a.heads * units;
    for (int64_t i = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; i < n; i += int64_t(gridDim.x) * blockDim.x) {
        const int u = int(i % units);
        const int64_t row = i / units;
        const int h = int(row % a.heads), t = int(row / a.heads);
        const int p = a.positions[t];
        const float *table = p >= 0 && p < a.max_positions ? a.table + int64_t(p) * a.rot : nullptr;
        rotate_unit<T, INTERLEAVED, VEC>(static_cast<const T *>(a.x) + t * a.x_token + h * a.x_head,
                                         static_cast<T *>(a.y) + t * a.y_token + h * a.y_head, table, u, a.dim, a.rot, sign);
    }
}

}  // namespace ffnrm::kv
