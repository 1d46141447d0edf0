// Attention over the 8-bit paged cache. A row (token t at position p, query head h) of sequence
// b sees the keys j < length with j <= p (causal) and j > p - window (window > 0):
//   y_j = scale * (q . kq_j) * sk_j,  out = sum_j softmax(y)_j * sv_j * vq_j
// with kq, vq the codes and sk, sv their pages' scales. One pass with a running maximum:
//   z_j = y_j log2(e) + log2(sv_j),  p_j = 2^(z_j - m) <= 1,  l = sum p_j / sv_j,
//   O = sum p_j vq_j,  out = O / l
// so the value scale costs nothing per element and the weights of the codes stay in (0, 1]. A
// row that sees no key gives zeros and lse = -inf.
#pragma once

#include "kv_common.cuh"

namespace ffnrm::kv {

struct AttendArgs {
    Pool pool;
    Batch batch;
    const void *q;
    void *out;
    float *lse;  // [rows][q_heads], or nullptr
    int64_t q_token, q_head, o_token, o_head;  // strides in elements
    int group;   // q heads per kv head
    float scale;
    int causal, window;
    int *status;
};

// One warp per (row, q head), keys in blocks of 32.
template <typename T, int D>
__global__ void __launch_bounds__(128) attend_rows_kernel(AttendArgs a) {
    constexpr float kLog2e = 1.4426950408889634f;
    const Pool &pl = a.pool;
    __shared__ float qs[4][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t item = blockIdx.x * 4ll + warp;
    const int heads = pl.heads * a.group;
    if (item >= int64_t(a.batch.rows) * heads) return;
    const int row = int(item / heads), hq = int(item % heads), h = hq / a.group;
    const int s = a.batch.starts ? seq_of_row(a.batch.starts, a.batch.seqs, row) : row;
    int first, n, length;
    const bool ok = seq_rows(a.batch, s, first, n) & seq_length(a.batch, s, pl.page_shift, length);
    if (!ok || (length > 0 && length < n)) {
        if (lane == 0) atomicOr(a.status, kStatusLength);
        length = 0;
    }
    const bool mine = ok && row >= first && row < first + n;
    const int pos = length - n + row - first;
    const int hi = !mine ? 0 : a.causal ? min(length, pos + 1) : length;
    const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const T *q = static_cast<const T *>(a.q) + row * a.q_token + hq * a.q_head;
    for (int d = lane; d < D; d += 32) qs[warp][d] = to_f32(q[d]);
    __syncwarp();
    float m = -__int_as_float(0x7f800000), l = 0.f, o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = 0.f;
    for (int j0 = lo & ~31; j0 < hi; j0 += 32) {
        const int j = j0 + lane;
        const bool seen = j >= lo && j < hi;
        int page = -1;
        if (seen) page = a.batch.tables[int64_t(s) * a.batch.width + (j >> pl.page_shift)];
        const bool valid = page >= 0 && page < pl.pages;
        if (seen && !valid) atomicOr(a.status, kStatusPage);
        const int64_t ph = valid ? int64_t(page) * pl.heads + h : 0;
        const int64_t at = (ph * pl.page_tokens + (j & (pl.page_tokens - 1))) * D;
        float z = -__int_as_float(0x7f800000), inv = 0.f;
        if (seen && valid) {
            float dot = 0.f;
            for (int d = 0; d < D; d += 16) {
                const Vec<int8_t, 16> c = *reinterpret_cast<const Vec<int8_t, 16> *>(pl.k_codes + at + d);
#pragma unroll
                for (int i = 0; i < 16; ++i) dot = fmaf(qs[warp][d + i], float(c.v[i]), dot);
            }
            const float sv = pl.v_scale[ph];
            z = dot * (a.scale * kLog2e * pl.k_scale[ph]) + __log2f(sv);
            inv = __fdividef(1.f, sv);
        }
        float top = z;
        for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        const float to = fmaxf(m, top);
        const float base = to == -__int_as_float(0x7f800000) ? 0.f : to;
        const float fix = exp2f(m - base);
        const float p = seen && valid ? exp2f(z - base) : 0.f;
        m = to;
        l = l * fix + p * inv;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] *= fix;
        for (int k = 0; k < 32; ++k) {
            const float pk = __shfl_sync(0xffffffffu, p, k);
            const int64_t vk = __shfl_sync(0xffffffffu, at, k);
            if (__shfl_sync(0xffffffffu, int(seen && valid), k)) {
#pragma unroll
                for (int i = 0; i < D / 32; ++i) o[i] = fmaf(pk, float(pl.v_codes[vk + i * 32 + lane]), o[i]);
            }
        }
    }
    for (int k = 16; k; k >>= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
    T *out = static_cast<T *>(a.out) + row * a.o_token + hq * a.o_head;
    const float norm = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) out[i * 32 + lane] = from_f32<T>(o[i] * norm);
    if (a.lse && lane == 0) a.lse[item] = l == 0.f ? -__int_as_float(0x7f800000) : (m + log2f(l)) * 0.6931471805599453f;
}

}  // namespace ffnrm::kv
