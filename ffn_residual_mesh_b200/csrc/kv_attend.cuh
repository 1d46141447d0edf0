// Attention over the 8-bit paged cache. A row (token t at position p, query head h) of sequence
// b sees the keys j < length with j <= p (causal) and j > p - window (window > 0):
//   y_j = scale * (q . kq_j) * sk_j,  out = sum_j softmax(y)_j * sv_j * vq_j
// with kq, vq the codes and sk, sv their pages' scales. One pass with a running maximum:
//   z_j = y_j log2(e) + log2(sv_j),  p_j = 2^(z_j - m) <= 1,  l = sum p_j / sv_j,
//   O = sum p_j vq_j,  out = O / l
// so the value scale costs nothing per element and the weights of the codes stay in (0, 1]. A
// row that sees no key gives zeros and lse = -inf.
//
// The logarithm and 1 / sv need sv well inside f32. A block with sv below kLeastScale holds values of
// zero: it takes part with codes of zero under kZeroScale instead, so its keys keep their weight in l.
// (kZeroScale is near the quantiser's floor of 1e-12, so such a block moves neither the maximum nor
// the other blocks' p; with p = 2^-126 the smallest kept, l has weights down to 2^-86 against value scales of 1.)
#pragma once

#include "kv_common.cuh"

namespace ffnrm::kv {

constexpr float kLeastScale = 0x1p-64f, kZeroScale = 0x1p-40f;
// 1 / sv; the fast division gives 0 from 2^126 on, so it works on a quarter.
__device__ __forceinline__ float inverse_scale(float sv) { return 0.25f * __fdividef(1.f, 0.25f * sv); }
// Whether a block's values count as zero (a NaN or negative scale does not).
__device__ __forceinline__ bool zero_block(float sv) { return fabsf(sv) < kLeastScale; }

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

// Rows that belong to no sequence (before starts[0], from starts[seqs] on) become zeros.
template <typename T>
__device__ __forceinline__ void zero_loose_rows(const AttendArgs &a) {
    if (!a.batch.starts) return;
    const int lo = min(max(a.batch.starts[0], 0), a.batch.rows), hi = min(max(a.batch.starts[a.batch.seqs], 0), a.batch.rows);
    const int heads = a.pool.heads * a.group, loose = lo + a.batch.rows - max(lo, hi);
    for (int i = blockIdx.x; i < loose; i += gridDim.x) {
        const int row = i < lo ? i : max(lo, hi) + i - lo;
        for (int e = threadIdx.x; e < heads * a.pool.dim; e += blockDim.x)
            static_cast<T *>(a.out)[row * a.o_token + e / a.pool.dim * a.o_head + e % a.pool.dim] = from_f32<T>(0.f);
        if (a.lse)
            for (int h = threadIdx.x; h < heads; h += blockDim.x) a.lse[int64_t(row) * heads + h] = -__int_as_float(0x7f800000);
    }
}

}  // namespace ffnrm::kv
