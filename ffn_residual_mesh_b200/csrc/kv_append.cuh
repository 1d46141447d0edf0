// Appending to the 8-bit paged cache, and reading it back.
//
// A page holds page_tokens tokens of a sequence; its codes share one scale per head. For each
// (page, head) that receives new tokens
//   s_old = the scale if the page already holds earlier tokens of the sequence, else 0
//   s     = max(s_old, max|x_new| / 127, 1e-12)
// earlier codes become rint(q * (s_old / s)) and new ones rint(x / s) in [-127, 127], with IEEE
// division, round-half-even and the 1e-12 floor of the groupwise activation quantiser
// (scripts/benchmark_exact_radix_split_pipeline.py:39-47). A NaN or infinity among the new
// values makes the scale NaN, so it reaches every row that reads the page; so does an s_old that is
// no scale (negative, infinite or NaN). Keys are rotated in f32 before they are quantised.
//
// Bound by issue slots (rotation, two looks at a value, the quotient) and by the chain of dependent loads
// before the values: 11.5k tokens of 8 kv heads x 128 with 32 heads of q, bf16: 65 us (3.7 TB/s);
// 64 single tokens: 8.2 us. Reading them back in f32: 28 us (4.3 TB/s). The half layout's 16-byte path spills some of its
// 64 registers (append and read together, times their floor: 1.73 in half layout, 1.58 interleaved).
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

// Channels d0 .. d0+7 of one row in f32, rotated when `table` (the position's row) is given. VEC: rows
// and table in 16-byte accesses, the rotated part a multiple of 8 channels (16 in the half layout).
template <typename T, bool VEC, bool INTERLEAVED>
__device__ __forceinline__ void load_channels(const T *x, int d0, const float *table, int rot, float (&f)[8]) {
    auto run = [&](int d, float (&o)[8]) {
        if constexpr (VEC) {
            constexpr int N = 16 / sizeof(T);
#pragma unroll
            for (int j = 0; j < 8; j += N) {
                unpack<T, N>(*reinterpret_cast<const Vec<T, N> *>(x + d + j), o + j);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = to_f32(x[d + i]);
        }
    };
    run(d0, f);
    if (!table || d0 >= rot) return;
    const int half = rot / 2;
    if constexpr (VEC && INTERLEAVED) {
        float c[4], s[4];
        load_table(table + d0 / 2, c);
        load_table(table + half + d0 / 2, s);
#pragma unroll
        for (int i = 0; i < 4; ++i) rotate_pair(f[2 * i], f[2 * i + 1], c[i], s[i]);
    } else if constexpr (VEC) {
        const bool low = d0 < half;
        const int p0 = low ? d0 : d0 - half;
        float g[8], c[8], s[8];
        run(low ? d0 + half : p0, g);
        load_table(table + p0, c);
        load_table(table + half + p0, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float a = low ? f[i] : g[i], b = low ? g[i] : f[i];
            rotate_pair(a, b, c[i], s[i]);
            f[i] = low ? a : b;
        }
    } else {
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
            const int d = d0 + i;
            if (d >= rot) break;
            const bool first = INTERLEAVED ? d % 2 == 0 : d < half;
            const int p = INTERLEAVED ? d / 2 : first ? d : d - half;
            float a = to_f32(x[INTERLEAVED ? 2 * p : p]), b = to_f32(x[INTERLEAVED ? 2 * p + 1 : p + half]);
            rotate_pair(a, b, table[p], table[half + p]);
            const float r = first ? a : b;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k == i) f[k] = r;
        }
    }
}

// Eight codes rint(x / s), |x| <= 127 s, inv = 1 / s rounded to nearest. The quotient is rounded as IEEE
// division rounds it, by Markstein's correction: the remainder of a quotient within one ulp is exact in
// a fused multiply-add, and adding it times inv rounds correctly; the first of the two steps brings x inv
// within that ulp. (Ties are common: bf16 values over a bf16 maximum hit a half exactly once in some two
// hundred.) The rounding is the addition of 1.5 * 2^23, whose sum has the integer in its low byte.
__device__ __forceinline__ uint2 quantise(const float (&f)[8], float s, float inv) {
    uint32_t t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float y = f[i] * inv;
        y = fmaf(fmaf(-y, s, f[i]), inv, y);
        y = fmaf(fmaf(-y, s, f[i]), inv, y);
        t[i] = __float_as_uint(__fadd_rn(y, 12582912.f));
    }
    return make_uint2(__byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(t[4], t[5], 0x0040), __byte_perm(t[6], t[7], 0x0040), 0x5410));
}

constexpr int kQueryHeads = 4;  // heads of q that a thread rotates
constexpr int kKept = 2;        // rows (twice 8 channels) that a thread keeps between the two looks at the values

// Blocks [0, slots * heads * 2): one (page, head, K or V) each. The rest: rows of q, rotated to
// q_out, in runs of 256 units.
template <typename T, bool VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(256, 4) append_kernel(AppendArgs a) {
    const Pool &pl = a.pool;
    const int items = a.slots * pl.heads * 2;
    const int P = pl.page_tokens, D = pl.dim;
    if (int(blockIdx.x) >= items) {
        // one thread per unit of kQueryHeads heads of a row
        constexpr int N = VEC ? 16 / int(sizeof(T)) : 1;
        const int units = rotary_units<INTERLEAVED, N>(D, a.rot), per_row = units * ((a.q_heads + kQueryHeads - 1) / kQueryHeads);
        const int64_t i = int64_t(int(blockIdx.x) - items) * 256 + threadIdx.x;
        const int row = int(i / per_row), i0 = int(i - int64_t(row) * per_row), g = i0 / units, h = g * kQueryHeads;
        if (row >= a.batch.rows) return;
        int s = row;
        if (a.batch.starts) {
            s = 0;
            for (int hi = a.batch.seqs; hi - s > 1;) {
                const int mid = (s + hi) / 2;
                if (__ldg(a.batch.starts + mid) <= row) s = mid;
                else hi = mid;
            }
        }
        int first, n, length;
        const bool ok = seq_rows(a.batch, s, first, n) & seq_length(a.batch, s, pl.page_shift, length);
        const T *x = static_cast<const T *>(a.q) + row * a.q_token + h * a.q_head;
        T *y = static_cast<T *>(a.q_out) + row * a.o_token + h * a.o_head;
        if (!ok || row < first || row >= first + n || length == 0 || length < n) {  // an idle row: zeros
            for (int k = 0; k < kQueryHeads && h + k < a.q_heads; ++k)
                for (int d = i0 - g * units; d < D; d += units) y[k * a.o_head + d] = from_f32<T>(0.f);
            return;
        }
        const int pos = length - n + row - first;
        const float *table = pos < a.max_positions ? a.table + int64_t(pos) * a.rot : nullptr;
        rotate_unit<T, INTERLEAVED, N, kQueryHeads>(x, y, a.q_head, a.o_head, a.q_heads - h, table, i0 - g * units, D, a.rot, 1.0f);
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
    const int base = block << pl.page_shift;
    const int lo = max(base, held), hi = min(base + P, length), old = max(0, held - base);
    const bool rotate = kv == 0 && a.table != nullptr, past = a.table && hi > a.max_positions;
    const T *x = static_cast<const T *>(kv ? a.v : a.k) + h * (kv ? a.v_head : a.k_head);
    const int64_t stride = kv ? a.v_token : a.k_token;
    // a thread's channels: d0 .. d0 + 7 and the same of the row's upper half
    const int per_row = D / 16, rows = 256 / per_row;
    const int d0 = int(threadIdx.x) % per_row * 8, d1 = d0 + D / 2, r0 = int(threadIdx.x) / per_row;
    auto values = [&](int p, float (&f)[2][8]) {
        const T *row = x + (first + p - held) * stride;
        const float *table = rotate ? a.table + int64_t(p) * a.rot : nullptr;
        if (VEC && !INTERLEAVED && table && a.rot == D) {  // the two runs are each other's pairs
            load_channels<T, VEC, INTERLEAVED>(row, d0, nullptr, 0, f[0]);
            load_channels<T, VEC, INTERLEAVED>(row, d1, nullptr, 0, f[1]);
            float c[8], s[8];
            load_table(table + d0, c);
            load_table(table + d1, s);
#pragma unroll
            for (int i = 0; i < 8; ++i) rotate_pair(f[0][i], f[1][i], c[i], s[i]);
        } else {
            load_channels<T, VEC, INTERLEAVED>(row, d0, table, a.rot, f[0]);
            load_channels<T, VEC, INTERLEAVED>(row, d1, table, a.rot, f[1]);
        }
    };
    // The first kKept rows stay in registers (a whole page of 64 x 128), their loads under way together
    // with the page's; the rest is read again.
    float kept[kKept][2][8];
    uint32_t bits = 0;  // the largest |x| as bits: infinities and NaN are above every number
    auto look = [&](const float (&f)[2][8]) {
#pragma unroll
        for (int i = 0; i < 16; ++i) bits = max(bits, __float_as_uint(f[i / 8][i % 8]) & 0x7fffffffu);
    };
    if (!past) {
#pragma unroll
        for (int k = 0; k < kKept; ++k)
            if (lo + r0 + k * rows < hi) values(lo + r0 + k * rows, kept[k]);
    }
    if (past || page < 0 || page >= pl.pages) {  // neither keys nor values of that page
        if (threadIdx.x == 0) atomicOr(a.status, past ? kStatusRotary : kStatusPage);
        return;
    }
    const int64_t ph = int64_t(page) * pl.heads + h;
    int8_t *codes = (kv ? pl.v_codes : pl.k_codes) + ph * P * D;
    float *scale = (kv ? pl.v_scale : pl.k_scale) + ph;
    const float before = old ? *scale : 0.f;  // thread 0 replaces it below the barriers
#pragma unroll
    for (int k = 0; k < kKept; ++k)
        if (lo + r0 + k * rows < hi) look(kept[k]);
    for (int p = lo + r0 + kKept * rows; p < hi; p += rows) {
        float f[2][8];
        values(p, f);
        look(f);
    }
    bits = __reduce_max_sync(0xffffffffu, bits);
    __shared__ uint32_t part[8];
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = bits;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) bits = max(bits, part[i]);
    const bool bad = bits >= 0x7f800000u || sound_scale(before) != before;
    const float fresh = bad ? __int_as_float(0x7fffffff) : fmaxf(fmaxf(before, __fdiv_rn(__uint_as_float(bits), 127.f)), 1e-12f);
    if (threadIdx.x == 0) *scale = fresh;
    if (!bad && old && fresh != before) {
        const float ratio = __fdiv_rn(before, fresh);
        for (int i = int(threadIdx.x) * 16; i < old * D; i += 256 * 16) {
            Vec<int8_t, 16> c = *reinterpret_cast<const Vec<int8_t, 16> *>(codes + i);
#pragma unroll
            for (int j = 0; j < 16; ++j) c.v[j] = int8_t(__float2int_rn(__fmul_rn(float(c.v[j]), ratio)));
            *reinterpret_cast<Vec<int8_t, 16> *>(codes + i) = c;
        }
    }
    const float inv = __frcp_rn(fresh);
    auto put = [&](int p, const float (&f)[2][8]) {
        int8_t *to = codes + (p - base) * D;
        *reinterpret_cast<uint2 *>(to + d0) = bad ? make_uint2(0u, 0u) : quantise(f[0], fresh, inv);
        *reinterpret_cast<uint2 *>(to + d1) = bad ? make_uint2(0u, 0u) : quantise(f[1], fresh, inv);
    };
#pragma unroll
    for (int k = 0; k < kKept; ++k)
        if (lo + r0 + k * rows < hi) put(lo + r0 + k * rows, kept[k]);
    for (int p = lo + r0 + kKept * rows; p < hi; p += rows) {
        float f[2][8];
        values(p, f);
        put(p, f);
    }
}

struct ReadArgs {
    Pool pool;
    Batch batch;
    void *k, *v;  // [rows][heads][dim]
    int *status;
};

// One warp per row: codes times scale, in the output type.
template <typename T>
__global__ void __launch_bounds__(256) read_kernel(ReadArgs a) {
    const Pool &pl = a.pool;
    const int row = int(blockIdx.x) * 8 + int(threadIdx.x >> 5), lane = threadIdx.x & 31, P = pl.page_tokens, D = pl.dim;
    if (row >= a.batch.rows) return;
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
    } else if (a.batch.starts && (row < a.batch.starts[0] || row >= a.batch.starts[a.batch.seqs])) {
        why = 0;  // and so does a row of no sequence
    }
    if (page < 0 && why && lane == 0) atomicOr(a.status, why);
    // 32 bytes of output (a whole sector) a lane: consecutive lanes along a head, then the heads
    constexpr int N = 32 / sizeof(T);
    const int per_head = D / N, count = pl.heads * per_head;
    const int64_t at = (int64_t(max(page, 0)) * pl.heads * P + (pos & (P - 1))) * D;
    const float none = why ? __int_as_float(0x7fffffff) : 0.f;
#pragma unroll 4
    for (int i = lane; i < 2 * count; i += 32) {
        const int kv = i >= count, r = kv ? i - count : i, h = r / per_head, d0 = r % per_head * N;
        Vec<int8_t, N> c{};
        float scale = none;
        if (page >= 0) {
            c = *reinterpret_cast<const Vec<int8_t, N> *>((kv ? pl.v_codes : pl.k_codes) + at + int64_t(h) * P * D + d0);
            scale = (kv ? pl.v_scale : pl.k_scale)[int64_t(page) * pl.heads + h];
        }
        float f[N];
#pragma unroll
        for (int k = 0; k < N; ++k) f[k] = __fmul_rn(float(c.v[k]), scale);
        union {
            Vec<T, N / 2> half[2];
            uint32_t u[8];
        } o{};
        o.half[0] = pack<T, N / 2>(f);
        o.half[1] = pack<T, N / 2>(f + N / 2);
        T *to = static_cast<T *>(kv ? a.v : a.k) + (int64_t(row) * pl.heads + h) * D + d0;
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"l"(to), "r"(o.u[0]), "r"(o.u[1]), "r"(o.u[2]), "r"(o.u[3]),
                     "r"(o.u[4]), "r"(o.u[5]), "r"(o.u[6]), "r"(o.u[7])
                     : "memory");
    }
}

}  // namespace ffnrm::kv
