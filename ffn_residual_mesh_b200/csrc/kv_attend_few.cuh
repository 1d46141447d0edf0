// Attention over the 8-bit paged cache for few query rows per sequence (single tokens, a few
// tokens): bound by reading the codes once, so the work is split over the keys.
//
// Rows of one kv head (tokens x group) sit on the N side of mma.sync m16n8k16 and 16 keys on the
// M side, for both products: S^T = K Q^T and O^T = V^T P^T. Codes go from global memory straight
// to the operand registers: a thread reads 16 contiguous channels of a key (and of four keys of V),
// and since the contracted index may be permuted as long as both operands agree, the bytes are
// in place as they come. int8 -> f16 is exact: byte ^ 0x80 under the exponent of 1024 gives
// 1152 + q, minus 1152 (leaving the bias in K's operand and starting S from -1152 sum q would save 32 of
// some 400 instructions per tile, but cost a logit 2e-5). S^T becomes P^T's operand by one 8x8
// transpose per 8 keys.
//
// The running maximum moves only when a score passes it by 2^8 (p stays below 2^15 in f16 with
// the 2^7 offset), which a vote per 16 keys decides.
//
// Bound by the issue slots of the conversion: 418 instructions for 16 keys x 128 channels, half of them
// widening int8 to f16, against HBM at 4.6 TB/s (24 contexts of up to 32k tokens, 8 kv heads x 128,
// 64 query heads: 358 MB in 76-79 us, 70% of the measured copy rate; one context of 131072: 67 us). Short contexts
// pay for the item itself, whose eight warps join through shared memory however few keys they had (39 contexts of
// up to 418 keys, 16 x 16 heads: 37 us for 3.5 us of bytes). At head dim 256 with 9 to 16 rows the kernel has 255
// registers, spills some and runs one block an SM (22 contexts of up to 846 keys: 57 us for 8.4 us of bytes).
//
// Work split: all (sequence, kv head, row tile) items, cut into units of 16 W keys, are laid on a
// line; each block takes an equal stretch of it. An item cut between blocks leaves partial
// (m, l, O) in the workspace, and the block that arrives last joins them in order.
#pragma once

#include <type_traits>

#include "kv_attend.cuh"

namespace ffnrm::kv {

constexpr float kFewOffset = 7.f, kFewStep = 8.f;
constexpr int kFewSeqs = 4096;  // most sequences of a call

__device__ __forceinline__ uint32_t hsub2_bits(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
// Bytes 0,1 (or 2,3) of w, biased by 128, as two f16 of the signed codes.
template <int HIGH>
__device__ __forceinline__ uint32_t codes_f16x2(uint32_t biased) {
    return hsub2_bits(__byte_perm(biased, 0x64646464u, HIGH ? 0x4342 : 0x4140), 0x64806480u);
}
__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint4 ldg_stream16(const int8_t *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 ldg_stream8(const int8_t *p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

// floor(a b / n) for the split of the line, in 32 bits where they are enough (a 64-bit division takes a
// tenth of a microsecond at the start of every block).
__device__ __forceinline__ int64_t share(int64_t a, int64_t b, int64_t n) {
    const uint64_t x = uint64_t(a) * uint64_t(b);
    if ((x | uint64_t(n)) >> 32 == 0) return uint32_t(x) / uint32_t(n);
    return int64_t(x / uint64_t(n));
}

struct FewArgs {
    AttendArgs a;
    float *partial;  // [2 * gridDim.x][rows of a tile][D + 2]
    int *counters;   // [gridDim.x], zero between calls
    int min_units;   // units that a block takes at least
    int most_rows;   // sequences with more rows belong to the other kernel
};

// The stretch of a sequence that its rows see, in units of UK keys, and its row tiles. On the line an item
// takes kFewItem units more, about what its queries, first loads and output cost beside the keys
// (without them a block with 18 short items ran three times as long as one with 50 units of one). Extra units of
// 1 / 3 / 6 / 10, us: 24 contexts of up to 32k tokens at head dim 128 85 / 77 / 79 / 82, 64 91 / 84 / 86 / 88, 256 103 / 92 / 97 /
// 100, in the 16-row variant 88 / 73 / 74 / 78; 256 contexts of up to 2048 100 / 89 / 101 / 113; 39 of up to 418 39 / 37 / 41 /
// 41; 22 of up to 846 at head dim 256 61 / 57 / 61 / 64; 16 x 5 tokens 59 / 42 / 45 / 51.
constexpr int kFewItem = 3;
struct SeqWork {
    int first, n, length, unit0, units, tiles;
    __device__ __forceinline__ int span() const { return units ? units + kFewItem : 0; }
};
template <int UK, int RT>
__device__ __forceinline__ SeqWork seq_work(const AttendArgs &a, int s, int most_rows) {
    SeqWork w{};
    const bool ok = seq_rows(a.batch, s, w.first, w.n) & seq_length(a.batch, s, a.pool.page_shift, w.length);
    if (!ok || (w.length > 0 && w.length < w.n)) {
        atomicOr(a.status, kStatusLength);
        w.length = 0;
    }
    if (w.n == 0 || w.n > most_rows / a.group) return w;
    const int lo = a.window > 0 ? max(0, w.length - w.n - a.window + 1) : 0;
    w.unit0 = lo / UK;
    w.units = max(1, (w.length + UK - 1) / UK - w.unit0);  // an idle slot's rows are written too
    w.tiles = (w.n * a.group + RT - 1) / RT;
    return w;
}

// Bytes of dynamic shared memory and floats of one partial.
template <int D, int NT, int W>
constexpr int few_smem() { return W * 8 * NT * (D + 2) * 4; }
// Blocks of W warps that an SM should hold: the keys under way are what the registers of its warps hold.
template <int D, int NT, int W>
constexpr int few_blocks() { return (D == 64 ? (NT == 1 ? 20 : 12) : D == 128 ? (NT == 1 ? 16 : 8) : 8) / W; }
template <int D, int NT>
__host__ __device__ constexpr int few_slot() { return 8 * NT * (D + 2); }

// The item's rows from the pieces that blocks b0 .. b1 left, in their order. (A call of its own, so that
// the loads under way here take no registers from the loop over the keys.)
template <typename T, int D, int NT, int W>
__device__ __noinline__ void join_pieces(const FewArgs &f, int b0, int b1, bool second, int h, int tile, int rows, int first) {
    constexpr int RT = 8 * NT, SLOT = few_slot<D, NT>(), GO = 8;  // pieces under way at a time
    const AttendArgs &a = f.a;
    const float ninf = -__int_as_float(0x7f800000);
    for (int e = threadIdx.x; e < rows * (D / 4); e += W * 32) {
        const int r = e / (D / 4), d = e % (D / 4) * 4;
        float top = ninf, sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int b = b0; b <= b1; b += GO) {
            float mk[GO], lk[GO];
            float4 x[GO];
#pragma unroll
            for (int i = 0; i < GO; ++i) {
                // block b0 may have worked on another item before; every other one begins with this one
                const int at = min(b + i, b1);
                const float *p = f.partial + int64_t(2 * at + (at == b0 && second ? 1 : 0)) * SLOT;
                mk[i] = __ldcg(p + RT * D + r);
                lk[i] = __ldcg(p + RT * D + RT + r);
                x[i] = __ldcg(reinterpret_cast<const float4 *>(p + r * D + d));
            }
#pragma unroll
            for (int i = 0; i < GO; ++i) {
                if (b + i > b1) break;
                const float to = fmaxf(top, mk[i]);
                const float fa = top == ninf ? (sum != sum ? 1.f : 0.f) : ex2(top - to);
                const float fb = mk[i] == ninf ? (lk[i] != lk[i] ? 1.f : 0.f) : ex2(mk[i] - to);
                acc.x = acc.x * fa + x[i].x * fb;
                acc.y = acc.y * fa + x[i].y * fb;
                acc.z = acc.z * fa + x[i].z * fb;
                acc.w = acc.w * fa + x[i].w * fb;
                sum = sum * fa + lk[i] * fb;
                top = to;
            }
        }
        const int q = tile * RT + r, token = q / a.group, hq = h * a.group + q - token * a.group;
        const float norm = sum == 0.f ? 0.f : 1.f / sum;
        Vec<T, 4> y;
        y.v[0] = from_f32<T>(acc.x * norm), y.v[1] = from_f32<T>(acc.y * norm);
        y.v[2] = from_f32<T>(acc.z * norm), y.v[3] = from_f32<T>(acc.w * norm);
        *reinterpret_cast<Vec<T, 4> *>(static_cast<T *>(a.out) + (first + token) * a.o_token + hq * a.o_head + d) = y;
        if (a.lse && d == 0)
            a.lse[int64_t(first + token) * (a.pool.heads * a.group) + hq] =
                sum == 0.f ? ninf : (top - kFewOffset + lg2(sum)) * 0.6931471805599453f;
    }
}

template <typename T, int D, int NT, int W>
__global__ void __launch_bounds__(W * 32, few_blocks<D, NT, W>()) attend_few_kernel(const __grid_constant__ FewArgs f) {
    constexpr float kLog2e = 1.4426950408889634f;
    constexpr int RT = 8 * NT, UK = 16 * W, KV = D / 64, MT = D / 16, VB = D / 8;
    const AttendArgs &a = f.a;
    const Pool &pl = a.pool;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const float ninf = -__int_as_float(0x7f800000);
    extern __shared__ float smem[];  // [W][RT][D] partial O, then [W][RT] m, [W][RT] l
    float *sm_o = smem, *sm_m = smem + W * RT * D, *sm_l = sm_m + W * RT;
    __shared__ int s_last;

    zero_loose_rows<T>(a);
    // This block's stretch of the line of units.
    // (sequences in runs of 32; above one run the warps share them out and leave each run's sum)
    __shared__ int64_t run_sum[kFewSeqs / 32];
    const int runs = (a.batch.seqs + 31) / 32;
    auto span_of = [&](int s) -> int64_t {
        if (s >= a.batch.seqs) return 0;
        const SeqWork w = seq_work<UK, RT>(a, s, f.most_rows);
        return int64_t(w.span()) * w.tiles * pl.heads;
    };
    auto warp_sum = [&](int64_t u) {
        for (int o = 16; o; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
        return u;
    };
    int64_t total = 0, mine = 0;
    if (runs <= 1) {
        mine = span_of(lane);
        total = warp_sum(mine);
    } else {
        for (int r = warp; r < runs; r += W) {
            const int64_t sum = warp_sum(span_of(r * 32 + lane));
            if (lane == 0) run_sum[r] = sum;
        }
        __syncthreads();
        for (int r = lane; r < runs; r += 32) total += run_sum[r];
        total = warp_sum(total);
    }
    if (total == 0) return;
    const int64_t blocks = min(int64_t(gridDim.x), share(total + f.min_units - 1, 1, f.min_units));
    if (blockIdx.x >= blocks) return;
    int64_t at = share(total, blockIdx.x, blocks);
    const int64_t end = share(total, blockIdx.x + 1, blocks), start = at;
    int64_t seq_at = 0;  // line position of sequence s
    int run = 0;
    if (runs > 1) {
        for (; run + 1 < runs && seq_at + run_sum[run] <= at; ++run) seq_at += run_sum[run];
        mine = span_of(run * 32 + lane);
    }
    int64_t upto = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    const unsigned past = __ballot_sync(0xffffffffu, seq_at + upto > at);
    const int who = past ? __ffs(past) - 1 : 0;
    int s = run * 32 + who;
    seq_at += __shfl_sync(0xffffffffu, upto - mine, who);

    while (at < end && s < a.batch.seqs) {
        const SeqWork w = seq_work<UK, RT>(a, s, f.most_rows);
        const int64_t item = w.units ? share(at - seq_at, 1, w.span()) : 0;
        if (w.units == 0 || item >= int64_t(w.tiles) * pl.heads) {
            seq_at += int64_t(w.span()) * w.tiles * pl.heads;
            ++s;
            continue;
        }
        const int h = int(share(item, 1, w.tiles)), tile = int(item - int64_t(h) * w.tiles);
        const int64_t item_at = seq_at + item * w.span(), item_end = item_at + w.span();
        const int u0 = max(0, int(at - item_at) - kFewItem), u1 = int(min(item_end, end) - item_at) - kFewItem;
        if (u1 <= u0) {  // the block's stretch ends before the item's first key
            at = min(item_end, end);
            continue;
        }
        const int rows = min(RT, w.n * a.group - tile * RT), pos0 = w.length - w.n;
        const int32_t *table = a.batch.tables + int64_t(s) * a.batch.width;

        const int token_lo = tile * RT / a.group, token_hi = (tile * RT + rows - 1) / a.group;
        // keys that every row of the tile sees: [all_lo, all_hi); that any sees: [any_lo, any_hi)
        const int any_hi = a.causal ? min(w.length, pos0 + token_hi + 1) : w.length;
        const int all_hi = a.causal ? min(w.length, pos0 + token_lo + 1) : w.length;
        const int any_lo = a.window > 0 ? max(0, pos0 + token_lo - a.window + 1) : 0;
        const int all_lo = a.window > 0 ? max(0, pos0 + token_hi - a.window + 1) : 0;

        auto key_of = [&](int u) { return (w.unit0 + u) * UK + warp * 16; };
        auto needed = [&](int u) { return u < u1 && key_of(u) < any_hi && key_of(u) + 16 > any_lo; };
        auto page_of = [&](int u) { return needed(u) ? table[key_of(u) >> pl.page_shift] : -1; };
        const int page = page_of(u0);
        int next_page = page_of(u0 + 1);  // on their way while the queries are read

        // queries: B operands, and per row the position and the scale
        uint32_t qb[NT][D / 16][2];
        float qs[NT][2];
        int qp[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = tile * RT + n * 8 + g;
            const bool live = n * 8 + g < rows;
            const int token = live ? r / a.group : 0, head = live ? r - token * a.group : 0;
            const T *q = static_cast<const T *>(a.q) + int64_t(w.first + token) * a.q_token + int64_t(h * a.group + head) * a.q_head;
            float v[D / 4];
#pragma unroll
            for (int j = 0; j < KV; ++j) {
                Vec<T, 16> x{};
                if (live) {
                    *reinterpret_cast<uint4 *>(&x.v[0]) = *reinterpret_cast<const uint4 *>(q + j * 64 + t * 16);
                    *reinterpret_cast<uint4 *>(&x.v[8]) = *reinterpret_cast<const uint4 *>(q + j * 64 + t * 16 + 8);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) v[j * 16 + i] = to_f32(x.v[i]);
            }
            float shift = 1.f;
            if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value) {
                // bf16 reaches past f16: the row is brought to [1, 2) by a power of two
                float m = 0.f;
#pragma unroll
                for (int i = 0; i < D / 4; ++i) m = fmaxf(m, fabsf(v[i]));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                const int e = min(max(int(__float_as_uint(m) >> 23), 1), 253);
                shift = __uint_as_float(uint32_t(e) << 23);
                const float down = __uint_as_float(uint32_t(254 - e) << 23);
#pragma unroll
                for (int i = 0; i < D / 4; ++i) v[i] *= down;
            }
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                qb[n][k][0] = pack_f16x2(v[4 * k], v[4 * k + 1]);
                qb[n][k][1] = pack_f16x2(v[4 * k + 2], v[4 * k + 3]);
            }
            // rows 2t, 2t+1 of the tile belong to lanes with g = 2t, 2t+1
            const float sc = shift * (a.scale * kLog2e);
            const int ps = pos0 + token;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                qs[n][i] = __shfl_sync(0xffffffffu, sc, (2 * t + i) * 4);
                qp[n][i] = __shfl_sync(0xffffffffu, ps, (2 * t + i) * 4);
            }
        }
        float o[MT][NT][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = ninf;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < MT; ++i) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
        }

        // A tile of 16 keys in registers: K words of keys g and g + 8, V words of keys 2t, 2t + 1, 2t + 8,
        // 2t + 9. Each half is loaded again as soon as its product has used it.
        uint32_t xk[KV][2][4], xv[4][VB / 4];
        float ks = 0.f, vs = 1.f;
        auto valid = [&](int u, int page) {  // keys without a page are left out
            const bool have = unsigned(page) < unsigned(pl.pages);
            if (!have && needed(u) && lane == 0) atomicOr(a.status, kStatusPage);
            return have;
        };
        auto load_k = [&](int u, int page) {
            const int64_t ph = int64_t(page) * pl.heads + h;
            const int8_t *kp = pl.k_codes + (ph * pl.page_tokens + (key_of(u) & (pl.page_tokens - 1))) * D + g * D + t * 16;
#pragma unroll
            for (int j = 0; j < KV; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint4 y = ldg_stream16(kp + i * 8 * D + j * 64);
                    xk[j][i][0] = y.x, xk[j][i][1] = y.y, xk[j][i][2] = y.z, xk[j][i][3] = y.w;
                }
        };
        auto load_v = [&](int u, int page) {
            const int64_t ph = int64_t(page) * pl.heads + h;
            const int8_t *vp = pl.v_codes + (ph * pl.page_tokens + (key_of(u) & (pl.page_tokens - 1))) * D + (2 * t) * D + g * (VB < 16 ? VB : 16);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int8_t *p = vp + (r & 1) * D + (r >> 1) * 8 * D;
                if constexpr (VB == 8) {
                    const uint2 y = ldg_stream8(p);
                    xv[r][0] = y.x, xv[r][1] = y.y;
                } else {
#pragma unroll
                    for (int j = 0; j < VB / 16; ++j) {
                        const uint4 y = ldg_stream16(p + j * 128);
                        xv[r][4 * j] = y.x, xv[r][4 * j + 1] = y.y, xv[r][4 * j + 2] = y.z, xv[r][4 * j + 3] = y.w;
                    }
                }
            }
            ks = pl.k_scale[ph];
            vs = pl.v_scale[ph];
        };
        bool have = valid(u0, page);
        if (have) {
            load_k(u0, page);
            load_v(u0, page);
        }
        for (int u = u0; u < u1; ++u) {
            const bool next = valid(u + 1, next_page);
            const int key = key_of(u), this_page = next_page;
            next_page = page_of(u + 2);
            if (!have) {
                have = next;
                if (next) {
                    load_k(u + 1, this_page);
                    load_v(u + 1, this_page);
                }
                continue;
            }
            have = next;
            // S^T = K Q^T: 16 keys x 8 NT rows
            float sc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
            for (int j = 0; j < KV; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t y = xk[j][0][k] ^ 0x80808080u, z = xk[j][1][k] ^ 0x80808080u;
                    const uint32_t a0 = codes_f16x2<0>(y), a1 = codes_f16x2<0>(z), a2 = codes_f16x2<1>(y), a3 = codes_f16x2<1>(z);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma16816(sc[n], a0, a1, a2, a3, qb[n][j * 4 + k][0], qb[n][j * 4 + k][1]);
                }
            if (next) load_k(u + 1, this_page);
            // z = y log2(e) + log2(sv); sc[n][i + 2 k]: key + g + 8 k, row 2t + i. A NaN value scale reaches the
            // rows that see it through its logarithm; it must not meet the others' p = 0.
            // (One test for all unusual scales, which the page's whole warp takes alike.)
            if (__float_as_uint(ks) >= 0x7f800000u || !(vs >= kLeastScale)) {
                ks = sound_scale(ks);
                if (zero_block(vs)) {
                    vs = kZeroScale;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int c = 0; c < VB / 4; ++c) xv[r][c] = 0;
                }
            }
            const float vlog = lg2(vs), vinv = vs == vs ? inverse_scale(vs) : 0.f;
            const bool whole = key + 16 <= all_hi && key >= all_lo;
            bool raise = false;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float f0 = qs[n][i] * ks;
#pragma unroll
                    for (int k = 0; k < 2; ++k) sc[n][i + 2 * k] = fmaf(sc[n][i + 2 * k], f0, vlog);
                }
            if (!whole) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int j = key + g + 8 * (i >> 1), p = qp[n][i & 1];
                        const bool seen = j < w.length && (!a.causal || j <= p) && (a.window <= 0 || j > p - a.window);
                        sc[n][i] = seen ? sc[n][i] : ninf;
                    }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) raise |= fmaxf(sc[n][i], sc[n][i + 2]) > m[n][i] + kFewStep;
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float top = fmaxf(sc[n][i], sc[n][i + 2]);
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        top = fmaxf(top, m[n][i]);
                        const float fix = m[n][i] == ninf ? 0.f : ex2(m[n][i] - top);
                        m[n][i] = top;
                        l[n][i] *= fix;
#pragma unroll
                        for (int c = 0; c < MT; ++c) {
                            o[c][n][i] *= fix;
                            o[c][n][i + 2] *= fix;
                        }
                    }
            }
            uint32_t pb[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float p[4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float base = m[n][i] == ninf ? 0.f : m[n][i] - kFewOffset;  // no key seen yet: 2^-inf = 0
                    p[i] = ex2(sc[n][i] - base);
                    p[i + 2] = ex2(sc[n][i + 2] - base);
                    l[n][i] = fmaf(p[i] + p[i + 2], vinv, l[n][i]);
                }
                pb[n][0] = transpose8x8(pack_f16x2(p[0], p[1]));
                pb[n][1] = transpose8x8(pack_f16x2(p[2], p[3]));
            }
            // O^T += V^T P^T: channels (thread g: 16 g + ..) x rows, over the 16 keys
#pragma unroll
            for (int c = 0; c < VB / 4; ++c) {  // 4 channels each
                const uint32_t lo01 = __byte_perm(xv[0][c], xv[1][c], 0x5140) ^ 0x80808080u, lo23 = __byte_perm(xv[0][c], xv[1][c], 0x7362) ^ 0x80808080u;
                const uint32_t hi01 = __byte_perm(xv[2][c], xv[3][c], 0x5140) ^ 0x80808080u, hi23 = __byte_perm(xv[2][c], xv[3][c], 0x7362) ^ 0x80808080u;
                const uint32_t a0 = codes_f16x2<0>(lo01), a1 = codes_f16x2<1>(lo01), a2 = codes_f16x2<0>(hi01), a3 = codes_f16x2<1>(hi01);
                const uint32_t b0 = codes_f16x2<0>(lo23), b1 = codes_f16x2<1>(lo23), b2 = codes_f16x2<0>(hi23), b3 = codes_f16x2<1>(hi23);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma16816(o[2 * c][n], a0, a1, a2, a3, pb[n][0], pb[n][1]);
                    mma16816(o[2 * c + 1][n], b0, b1, b2, b3, pb[n][0], pb[n][1]);
                }
            }
            if (next) load_v(u + 1, this_page);
        }

        // Join the warps. Row r's sums over the keys are spread over g.
        __syncthreads();  // the previous piece's reads of shared memory are done
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float x = l[n][i];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                const int r = n * 8 + 2 * t + i;
                if (g == 0) {
                    sm_m[warp * RT + r] = m[n][i];
                    sm_l[warp * RT + r] = x;
                }
                float *dst = sm_o + (warp * RT + r) * D;
                // m-tile c holds channels 2c, 2c + 1 of this thread's run (runs of 16, or 8 for D = 64)
#pragma unroll
                for (int c = 0; c < MT; ++c) {
                    const int d = VB == 8 ? g * 8 + 2 * c : (c / 8) * 128 + g * 16 + 2 * (c % 8);
                    *reinterpret_cast<float2 *>(dst + d) = make_float2(o[c][n][i], o[c][n][i + 2]);
                }
            }
        __syncthreads();
        const bool split = u0 > 0 || u1 < w.units;
        constexpr int SLOT = RT * (D + 2);
        const int slot = 2 * int(blockIdx.x) + (at == start ? 0 : 1);
        for (int e = tid; e < RT * (D / 4); e += W * 32) {
            const int r = e / (D / 4), d = e % (D / 4) * 4;
            if (r >= rows) continue;
            float top = ninf;
#pragma unroll
            for (int k = 0; k < W; ++k) top = fmaxf(top, sm_m[k * RT + r]);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < W; ++k) {
                const float mk = sm_m[k * RT + r];
                const float fix = mk == ninf ? (sm_l[k * RT + r] != sm_l[k * RT + r] ? 1.f : 0.f) : ex2(mk - top);
                const float4 x = *reinterpret_cast<const float4 *>(sm_o + (k * RT + r) * D + d);
                acc.x = fmaf(x.x, fix, acc.x);
                acc.y = fmaf(x.y, fix, acc.y);
                acc.z = fmaf(x.z, fix, acc.z);
                acc.w = fmaf(x.w, fix, acc.w);
                sum = fmaf(sm_l[k * RT + r], fix, sum);
            }
            if (split) {
                float *p = f.partial + int64_t(slot) * SLOT;
                __stcg(reinterpret_cast<float4 *>(p + r * D + d), acc);
                if (d == 0) {
                    __stcg(p + RT * D + r, top);
                    __stcg(p + RT * D + RT + r, sum);
                }
                continue;
            }
            const int q = tile * RT + r, token = q / a.group, hq = h * a.group + q - token * a.group;
            const float norm = sum == 0.f ? 0.f : 1.f / sum;
            Vec<T, 4> y;
            y.v[0] = from_f32<T>(acc.x * norm), y.v[1] = from_f32<T>(acc.y * norm);
            y.v[2] = from_f32<T>(acc.z * norm), y.v[3] = from_f32<T>(acc.w * norm);
            *reinterpret_cast<Vec<T, 4> *>(static_cast<T *>(a.out) + (w.first + token) * a.o_token + hq * a.o_head + d) = y;
            if (a.lse && d == 0)
                a.lse[int64_t(w.first + token) * (pl.heads * a.group) + hq] =
                    sum == 0.f ? ninf : (top - kFewOffset + lg2(sum)) * 0.6931471805599453f;
        }
        if (split) {
            // blocks that hold a piece of this item: unit u lies in block floor(((u + 1) blocks - 1) / total)
            const int b0 = int(((item_at + kFewItem + 1) * blocks - 1) / total), b1 = int((item_end * blocks - 1) / total);
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const int n = atomicAdd(f.counters + b0, 1);
                s_last = n == b1 - b0;
                if (s_last) f.counters[b0] = 0;
            }
            __syncthreads();
            if (s_last) {
                __threadfence();
                join_pieces<T, D, NT, W>(f, b0, b1, share(total, b0, blocks) < item_at, h, tile, rows, w.first);
            }
        }
        at = min(item_end, end);
    }
}

}  // namespace ffnrm::kv
