// Appending to the 8-bit paged cache, and reading it back.
//
// A page holds page_tokens tokens of a sequence; its codes share one scale per head. For each
// (page, head) that receives new tokens
//   s_old = the scale if the page already holds earlier tokens of the sequence, else 0
//   s     = max(s_old, max|x_new| / 127, 1e-12)
// earlier codes become rint(q * (s_old / s)) and new ones rint(x / s) in [-127, 127], with IEEE
// division, round-half-even and the 1e-12 floor of the groupwise activation quantiser
// (scripts/benchmark_exact_radix_split_pipeline.py:39-47). A NaN or infinity among the new
// values makes the scale NaN, so it reaches every row that reads the page. Keys are rotated
// in f32 before they are quantised.
#pragma once

#include "kv_common.cuh"
#include "kv_rotary.cuh"

namespace ffnrm::kv {

struct AppendArgs {
    Pool pool;
    Batch batch;
    const void *k, *v, *q;
    void *q_out;
    int64_t k_token, k_head, v_token, v_head, q_token, q_head, o_token, o_head;  // strides in elements
    const float *table;  // nullptr: no rotation
    int rot, max_positions, q_heads;
    int slots;           // upper bound of the pages that receive tokens
    int q_chunks;        // blocks per row of q
    int *status;
};

// Slots of the work list: sequence s owns slots [starts[s]/P + 2s, starts[s+1]/P + 2(s+1)), at
// least as many as the pages its n tokens can touch ((n - 1)/P + 2), so no scan is needed.
__host__ __device__ inline int append_slots(int seqs, int rows, int page_shift, bool ragged) {
    return ragged ? (rows >> page_shift) + 2 * seqs : seqs;
}
__device__ __forceinline__ int seq_of_slot(const int32_t *starts, int seqs, int page_shift, int slot) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = seqs;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int probe = lo + lane * step;
        const unsigned m = __ballot_sync(0xffffffffu, probe < hi && (starts[probe] >> page_shift) + 2 * probe <= slot);
        const int last = m ? 31 - __clz(m) : 0;
        lo += last * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

// Channels d0 .. d0+7 of one row in f32, rotated when `table` (the position's row) is given.
template <typename T, bool VEC>
__device__ __forceinline__ void load_channels(const T *x, int d0, const float *table, int rot, bool interleaved, float (&f)[8]) {
    auto run = [&](int d, float (&o)[8]) {
        if constexpr (VEC) {
            constexpr int N = 16 / sizeof(T);
#pragma unroll
            for (int j = 0; j < 8; j += N) {
                const Vec<T, N> v = *reinterpret_cast<const Vec<T, N> *>(x + d + j);
#pragma unroll
                for (int i = 0; i < N; ++i) o[j + i] = to_f32(v.v[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = to_f32(x[d + i]);
        }
    };
    run(d0, f);
    if (!table || d0 >= rot) return;
    const int half = rot / 2;
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const int p = (d0 + i) / 2;
            if (p < half) rotate_pair(f[i], f[i + 1], table[p], table[half + p]);
        }
    } else if (half % 8 == 0) {
        float g[8];
        const bool low = d0 < half;
        run(low ? d0 + half : d0 - half, g);
        const int p0 = low ? d0 : d0 - half;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float c = table[p0 + i], s = table[half + p0 + i];
            float a = low ? f[i] : g[i], b = low ? g[i] : f[i];
            rotate_pair(a, b, c, s);
            f[i] = low ? a : b;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = d0 + i;
            if (d >= rot) break;
            const bool low = d < half;
            const int p = low ? d : d - half;
            float a = low ? f[i] : to_f32(x[p]), b = low ? to_f32(x[p + half]) : f[i];
            rotate_pair(a, b, table[p], table[half + p]);
            f[i] = low ? a : b;
        }
    }
}

__device__ __forceinline__ int quantise(float x, float s) {
    return max(-127, min(127, __float2int_rn(__fdiv_rn(x, s))));
}

// Blocks [0, slots * heads * 2): one (page, head, K or V) each. The rest: rows of q, rotated to
// q_out, in runs of 256 units.
template <typename T, bool VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(256) append_kernel(AppendArgs a) {
    const Pool &pl = a.pool;
    const int items = a.slots * pl.heads * 2;
    const int P = pl.page_tokens, D = pl.dim;
    if (int(blockIdx.x) >= items) {
        const int i = int(blockIdx.x) - items;
        const int row = i / a.q_chunks, chunk = i % a.q_chunks;
        const int s = a.batch.starts ? seq_of_row(a.batch.starts, a.batch.seqs, row) : row;
        int first, n, length;
        const bool ok = seq_rows(a.batch, s, first, n) & seq_length(a.batch, s, pl.page_shift, length);
        if (!ok || row < first || row >= first + n || length == 0 || length < n) {  // an idle row: zeros
            if (chunk == 0)
                for (int e = threadIdx.x; e < a.q_heads * D; e += 256)
                    static_cast<T *>(a.q_out)[row * a.o_token + e / D * a.o_head + e % D] = from_f32<T>(0.f);
            return;
        }
        const int pos = length - n + row - first;
        const float *table = pos < a.max_positions ? a.table + int64_t(pos) * a.rot : nullptr;
        constexpr int N = VEC ? 16 / int(sizeof(T)) : 1;
        const int units = rotary_units<INTERLEAVED, N>(D, a.rot);
        const int u = chunk * 256 + int(threadIdx.x);
        if (u >= units * a.q_heads) return;
        const int h = u / units;
        rotate_unit<T, INTERLEAVED, N>(static_cast<const T *>(a.q) + row * a.q_token + h * a.q_head,
                                       static_cast<T *>(a.q_out) + row * a.o_token + h * a.o_head, table, u - h * units, D,
                                       a.rot, 1.0f);
        return;
    }
    const int kv = int(blockIdx.x) & 1, h = (int(blockIdx.x) >> 1) % pl.heads, slot = (int(blockIdx.x) >> 1) / pl.heads;
    int s = slot, nth = 0;
    if (a.batch.starts) {
        s = seq_of_slot(a.batch.starts, a.batch.seqs, pl.page_shift, slot);
        nth = slot - ((a.batch.starts[s] >> pl.page_shift) + 2 * s);
    }
    int first, n, length;
    const bool rows_ok = seq_rows(a.batch, s, first, n), length_ok = seq_length(a.batch, s, pl.page_shift, length);
    if (!rows_ok || !length_ok || (length > 0 && length < n)) {
        if (threadIdx.x == 0) atomicOr(a.status, kStatusLength);
        return;
    }
    if (length == 0 || n == 0 || nth < 0) return;
    const int held = length - n, block = (held >> pl.page_shift) + nth;
    if (block > (length - 1) >> pl.page_shift) return;
    const int page = a.batch.tables[int64_t(s) * a.batch.width + block];
    if (page < 0 || page >= pl.pages) {
        if (threadIdx.x == 0) atomicOr(a.status, kStatusPage);
        return;
    }
    const int base = block << pl.page_shift;
    const int lo = max(base, held), hi = min(base + P, length), old = max(0, held - base);
    const bool rotate = kv == 0 && a.table != nullptr;
    if (a.table && hi > a.max_positions) {  // neither keys nor values of that page
        if (threadIdx.x == 0) atomicOr(a.status, kStatusRotary);
        return;
    }
    const T *x = static_cast<const T *>(kv ? a.v : a.k) + h * (kv ? a.v_head : a.k_head);
    const int64_t stride = kv ? a.v_token : a.k_token;
    const int64_t ph = int64_t(page) * pl.heads + h;
    int8_t *codes = (kv ? pl.v_codes : pl.k_codes) + ph * P * D;
    float *scale = (kv ? pl.v_scale : pl.k_scale) + ph;

    const int per_row = D / 8, rows = 256 / per_row;
    const int d0 = int(threadIdx.x) % per_row * 8, r0 = int(threadIdx.x) / per_row;
    float amax = 0.f;
    bool bad = false;
    for (int p = lo + r0; p < hi; p += rows) {
        float f[8];
        load_channels<T, VEC>(x + (first + p - held) * stride, d0, rotate ? a.table + int64_t(p) * a.rot : nullptr, a.rot,
                              INTERLEAVED, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float m = fabsf(f[i]);
            bad |= !(m < __int_as_float(0x7f800000));
            amax = fmaxf(amax, m);
        }
    }
    bad = __syncthreads_or(bad);
    for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    __shared__ float part[8];
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = amax;
    const float before = old ? *scale : 0.f;  // read before thread 0 replaces it, below the barrier
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, part[i]);
    bad |= before != before;
    const float fresh = bad ? __int_as_float(0x7fffffff) : fmaxf(fmaxf(before, __fdiv_rn(amax, 127.f)), 1e-12f);
    if (threadIdx.x == 0) *scale = fresh;
    if (!bad && old && fresh != before) {
        const float ratio = __fdiv_rn(before, fresh);
        for (int i = int(threadIdx.x) * 8; i < old * D; i += 256 * 8) {
            Vec<int8_t, 8> c = *reinterpret_cast<const Vec<int8_t, 8> *>(codes + i);
#pragma unroll
            for (int j = 0; j < 8; ++j) c.v[j] = int8_t(__float2int_rn(__fmul_rn(float(c.v[j]), ratio)));
            *reinterpret_cast<Vec<int8_t, 8> *>(codes + i) = c;
        }
    }
    for (int p = lo + r0; p < hi; p += rows) {
        float f[8];
        load_channels<T, VEC>(x + (first + p - held) * stride, d0, rotate ? a.table + int64_t(p) * a.rot : nullptr, a.rot,
                              INTERLEAVED, f);
        Vec<int8_t, 8> c;
#pragma unroll
        for (int i = 0; i < 8; ++i) c.v[i] = bad ? int8_t(0) : int8_t(quantise(f[i], fresh));
        *reinterpret_cast<Vec<int8_t, 8> *>(codes + (p - base) * D + d0) = c;
    }
}

struct ReadArgs {
    Pool pool;
    Batch batch;
    void *k, *v;  // [rows][heads][dim]
    int *status;
};

// One block per row: codes times scale, in the output type.
template <typename T>
__global__ void __launch_bounds__(256) read_kernel(ReadArgs a) {
    const Pool &pl = a.pool;
    const int row = blockIdx.x, P = pl.page_tokens, D = pl.dim;
    const int s = a.batch.starts ? seq_of_row(a.batch.starts, a.batch.seqs, row) : row;
    int first, n, length;
    const bool rows_ok = seq_rows(a.batch, s, first, n), length_ok = seq_length(a.batch, s, pl.page_shift, length);
    int page = -1, pos = 0, why = kStatusLength;
    if (rows_ok && length_ok && row >= first && row < first + n && length >= n) {
        pos = length - n + row - first;
        page = a.batch.tables[int64_t(s) * a.batch.width + (pos >> pl.page_shift)];
        if (page < 0 || page >= pl.pages) {
            page = -1;
            why = kStatusPage;
        }
    } else if (rows_ok && length_ok && length == 0) {
        why = 0;  // an idle slot reads as zeros
    }
    if (page < 0 && why && threadIdx.x == 0) atomicOr(a.status, why);
    const int per_head = D / 8;
    for (int i = threadIdx.x; i < 2 * pl.heads * per_head; i += 256) {
        const int kv = i / (pl.heads * per_head), r = i % (pl.heads * per_head), h = r / per_head, d0 = r % per_head * 8;
        Vec<int8_t, 8> c{};
        float scale = why ? __int_as_float(0x7fffffff) : 0.f;
        if (page >= 0) {
            const int64_t ph = int64_t(page) * pl.heads + h;
            c = *reinterpret_cast<const Vec<int8_t, 8> *>((kv ? pl.v_codes : pl.k_codes) + (ph * P + (pos & (P - 1))) * D + d0);
            scale = (kv ? pl.v_scale : pl.k_scale)[ph];
        }
        T *out = static_cast<T *>(kv ? a.v : a.k) + (int64_t(row) * pl.heads + h) * D + d0;
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int j = 0; j < 8; j += N) {
            Vec<T, N> o;
#pragma unroll
            for (int i2 = 0; i2 < N; ++i2) o.v[i2] = from_f32<T>(__fmul_rn(float(c.v[j + i2]), scale));
            *reinterpret_cast<Vec<T, N> *>(out + j) = o;
        }
    }
}

}  // namespace ffnrm::kv
