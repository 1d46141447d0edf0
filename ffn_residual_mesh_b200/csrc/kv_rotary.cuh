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

// Whether VEC channels at a time cover the row's halves and rest, and the table's rows allow 16-byte
// accesses.
inline bool rotary_fits(bool interleaved, int vec, int dim, int rot, const float *table) {
    return dim % vec == 0 && rot % 8 == 0 && (interleaved || (rot / 2) % vec == 0) && reinterpret_cast<uintptr_t>(table) % 16 == 0;
}

// N consecutive table entries, in 16-byte accesses where the alignment allows (N >= 4).
template <int N>
__device__ __forceinline__ void load_table(const float *p, float (&v)[N]) {
    if constexpr (N >= 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 x = __ldg(reinterpret_cast<const float4 *>(p + i));
            v[i] = x.x, v[i + 1] = x.y, v[i + 2] = x.z, v[i + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __ldg(p + i);
    }
}

// Rotates unit u of HEADS head rows (x, y: the first; they may be the same), the cosines and sines
// loaded once for all. `table` is the position's row, nullptr for a position outside the table: the
// rotated channels become NaN. Rows from `heads` on are left alone.
template <typename T, bool INTERLEAVED, int VEC, int HEADS>
__device__ __forceinline__ void rotate_unit(const T *x, T *y, int64_t x_head, int64_t y_head, int heads, const float *table, int u,
                                            int dim, int rot, float sign) {
    const int half = rot / 2;
    const int rotated = ((INTERLEAVED && VEC > 1) ? rot : half) / VEC;
    if (u >= rotated) {
        const int d = rot + (u - rotated) * VEC;
        Vec<T, VEC> v[HEADS];
#pragma unroll
        for (int h = 0; h < HEADS; ++h)
            if (h < heads) v[h] = *reinterpret_cast<const Vec<T, VEC> *>(x + h * x_head + d);
#pragma unroll
        for (int h = 0; h < HEADS; ++h)
            if (h < heads) *reinterpret_cast<Vec<T, VEC> *>(y + h * y_head + d) = v[h];
        return;
    }
    constexpr bool TOGETHER = INTERLEAVED && VEC > 1;  // both members of a pair in one access
    constexpr int PAIRS = TOGETHER ? VEC / 2 : VEC;
    const int ia = TOGETHER ? u * VEC : INTERLEAVED ? 2 * u : u * VEC, ib = INTERLEAVED ? 2 * u + 1 : u * VEC + half;
    Vec<T, VEC> va[HEADS], vb[HEADS];
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
        if (h < heads) {
            va[h] = *reinterpret_cast<const Vec<T, VEC> *>(x + h * x_head + ia);
            if constexpr (!TOGETHER) vb[h] = *reinterpret_cast<const Vec<T, VEC> *>(x + h * x_head + ib);
        }
    float c[PAIRS], s[PAIRS];
    if (table) {
        load_table(table + u * PAIRS, c);
        load_table(table + half + u * PAIRS, s);
    } else {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) c[i] = s[i] = __int_as_float(0x7fffffff);
    }
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        if (h >= heads) break;
        float fa[VEC], fb[VEC];
        unpack<T, VEC>(va[h], fa);
        if constexpr (!TOGETHER) unpack<T, VEC>(vb[h], fb);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            if constexpr (TOGETHER)
                rotate_pair(fa[2 * i], fa[2 * i + 1], c[i], sign * s[i]);
            else
                rotate_pair(fa[i], fb[i], c[i], sign * s[i]);
        }
        *reinterpret_cast<Vec<T, VEC> *>(y + h * y_head + ia) = pack<T, VEC>(fa);
        if constexpr (!TOGETHER) *reinterpret_cast<Vec<T, VEC> *>(y + h * y_head + ib) = pack<T, VEC>(fb);
    }
}

// One thread per unit of HEADS head rows. Bound by reading and writing x once (16384 x 32 x 128 bf16, half
// of it rotated: interleaved 53 us, 5.1 TB/s, 78% of the measured copy rate, one head to a thread 74 us; half layout 66 us): several rows under way per
// thread keep enough bytes in flight, and a table row is read once for HEADS heads.
template <typename T, bool INTERLEAVED, int VEC, int HEADS>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs a, float sign) {
    const unsigned units = rotary_units<INTERLEAVED, VEC>(a.dim, a.rot), groups = (a.heads + HEADS - 1) / HEADS;
    const int64_t i = blockIdx.x * int64_t(blockDim.x) + threadIdx.x;
    int t, g, u;
    if (i >> 32 == 0) {
        const unsigned row = unsigned(i) / units;
        u = int(unsigned(i) - row * units), t = int(row / groups), g = int(row - unsigned(t) * groups);
    } else {
        const int64_t row = i / units;
        u = int(i - row * units), t = int(row / groups), g = int(row - int64_t(t) * groups);
    }
    if (t >= a.tokens) return;
    const int p = a.positions[t], h = g * HEADS;
    const float *table = p >= 0 && p < a.max_positions ? a.table + int64_t(p) * a.rot : nullptr;
    rotate_unit<T, INTERLEAVED, VEC, HEADS>(static_cast<const T *>(a.x) + t * a.x_token + h * a.x_head,
                                            static_cast<T *>(a.y) + t * a.y_token + h * a.y_head, a.x_head, a.y_head, a.heads - h,
                                            table, u, a.dim, a.rot, sign);
}

}  // namespace ffnrm::kv
