// Attention over the 8-bit paged cache for many query rows per sequence (prompt chunks): bound by
// the tensor cores and the exponentials, so both products run on tcgen05 and the softmax beside
// them.
//
// One block holds NQ tiles of 128 rows (tokens x group of one kv head; f16, K-major, 128-byte
// swizzle) and walks over the keys in tiles of BN. Warp roles:
//   softmax warpgroups, one per row tile, one thread per row: read S from TMEM, write P = 2^(z-m)
//     as f16 over it, rescale O in TMEM when the maximum moved by more than 2^8;
//   converter warpgroup: codes from global memory to f16 K and V tiles in shared memory (exact:
//     byte ^ 0x80 under the exponent of 1024, minus 1152), two stages each, and the tile's scales;
//   one MMA warp: S = Q K^T (K-major operands) and O += P V (P from TMEM, V as it lies in the
//     cache, N-major).
// With two row tiles the tensor cores work on one while the other's softmax runs. MMAs of one
// thread execute in order, so S of the next key tile may be written over P right behind the product
// that reads it.
//
// Per 128 keys and 256 rows the products need 2048 cycles and the exponentials left to the MUFU 1792; the
// loop takes some 4200, the chain S - softmax - P - products with its hand-overs (116 cycles each) being
// longer than either. Measured: 8192-token prompt, 32/8 heads x 128, causal: 580-591 us, 930-948
// TFLOP/s (57% of the measured GEMM burst); 4096 tokens at head dim 256: 345-357 us. A block has its set-up, query tile,
// first conversion and output to itself (one block an SM): with four key tiles to a block they weigh most (a prompt
// of 1073 tokens, 16 x 16 heads: 167 us for 46 us of products).
#pragma once

#include <type_traits>

#include "kv_attend_few.cuh"
#include "sm100.cuh"

namespace ffnrm::kv {

using namespace ffnrm::sm100;

// Shared-memory matrix descriptor of an N-major tile with 128-byte swizzle: 64 channels (128 B) per
// key row, 8-key atoms of 1024 B, `lbo` bytes between blocks of 64 channels.
__device__ __forceinline__ uint64_t umma_desc_sw128_mn(uint32_t addr, uint32_t lbo) {
    uint64_t d = 0;
    d |= uint64_t((addr >> 4) & 0x3FFF);
    d |= uint64_t((lbo >> 4) & 0x3FFF) << 16;
    d |= uint64_t(1024 >> 4) << 32;
    d |= uint64_t(1) << 46;
    d |= uint64_t(2) << 61;
    return d;
}
// Waits for the phase of `parity`, asleep in hardware for up to about 10 us at a time, so that the waiting
// warps leave the issue slots to the softmax (hints of 0.2 to 10 us measured the same); gives up
// after some seconds.
__device__ __forceinline__ bool wait_phase(uint64_t *bar, uint32_t parity, int *err, int code) {
    for (int i = 0; i < 400000; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity), "r"(10000u)
            : "memory");
        if (ok) return true;
    }
    atomicExch(err, code);
    return false;
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}
// D[tmem] (+)= A[tmem] * B[smem], kind::f16.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// 2^x of two values on the FMA pipe: x = n + r with n the nearest integer (Cody and Waite's reduction),
// 2^r by the minimax polynomial of degree 4 on [-1/2, 1/2] (relative error 2.6e-6), n added to the
// exponent. Values below -125 give 2^-125.
__device__ __forceinline__ float2 ex2_poly(float2 x) {
    const float2 magic = make_float2(12582912.f, 12582912.f);  // 1.5 * 2^23
    x = make_float2(fmaxf(x.x, -125.f), fmaxf(x.y, -125.f));
    const float2 t = fadd2(x, magic);
    const float2 n = fadd2(t, make_float2(-12582912.f, -12582912.f));
    const float2 r = ffma2(n, make_float2(-1.f, -1.f), x);
    float2 p = ffma2(r, make_float2(9.570102207e-3f, 9.570102207e-3f), make_float2(5.591786280e-2f, 5.591786280e-2f));
    p = ffma2(p, r, make_float2(2.402474433e-1f, 2.402474433e-1f));
    p = ffma2(p, r, make_float2(6.931217909e-1f, 6.931217909e-1f));
    p = ffma2(p, r, make_float2(9.999992847e-1f, 9.999992847e-1f));
    return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23)),
                       __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23)));
}

template <int D>
struct Many {
    static constexpr int NQ = D == 256 ? 1 : 2;    // row tiles of 128
    static constexpr int BN = D == 256 ? 64 : 128; // keys per tile
    static constexpr int SB = D == 256 ? 2 : 1;    // S buffers per row tile
    static constexpr int ROWS = 128 * NQ;
    static constexpr int CONV = D == 256 ? 2 : 1;  // converter warpgroups
    static constexpr int THREADS = 128 * (NQ + CONV + 1);
    static constexpr int Q_BYTES = 128 * D * 2, KV_BYTES = BN * D * 2;
    static constexpr int CHUNKS = BN / 16;         // runs of keys with one scale
    static constexpr int SMEM = 1024 + NQ * Q_BYTES + 4 * KV_BYTES + 2 * CHUNKS * 16 + 256;
    static constexpr int EARLY = BN / 4 * 3 / 32 * 32;  // keys of P that are handed over first
    static constexpr int O_COL = 256;              // first TMEM column of O
    static constexpr bool REGS = D != 256;         // 512 threads: registers are moved to the softmax
};

struct ManyArgs {
    AttendArgs a;
    int slots;     // upper bound of row tiles per kv head
    int few_rows;  // sequences with at most this many rows belong to the other kernel
    int alone;     // the other kernel is not launched
};

// Row-tile slots: sequence s owns [starts[s] G / ROWS + s, starts[s+1] G / ROWS + s + 1), at least the
// tiles that its n G rows fill.
__host__ __device__ inline int64_t many_slots(int seqs, int rows, int group, int tile) { return int64_t(rows) * group / tile + seqs; }
__device__ __forceinline__ int seq_of_many(const int32_t *starts, int seqs, int group, int tile, int slot) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = seqs;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int probe = lo + lane * step;
        const unsigned m = __ballot_sync(0xffffffffu, probe < hi && int64_t(starts[probe]) * group / tile + probe <= slot);
        const int last = m ? 31 - __clz(m) : 0;
        lo += last * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

template <typename T, int D>
__global__ void __launch_bounds__(Many<D>::THREADS, 1) attend_many_kernel(ManyArgs args) {
    using C = Many<D>;
    constexpr int NQ = C::NQ, BN = C::BN, SB = C::SB, KB = D / 64;
    constexpr float kLog2e = 1.4426950408889634f;
    const AttendArgs &a = args.a;
    const Pool &pl = a.pool;
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0), wg = warp >> 2;  // uniform for the compiler too
    const float ninf = -__int_as_float(0x7f800000);

    if (args.alone) zero_loose_rows<T>(a);
    // This block's sequence, row tile and kv head.
    const int h = int(blockIdx.x) % pl.heads, slot = int(blockIdx.x) / pl.heads;
    int s = slot, nth = 0;
    if (a.batch.starts) {
        s = seq_of_many(a.batch.starts, a.batch.seqs, a.group, C::ROWS, slot);
        nth = slot - int(int64_t(a.batch.starts[s]) * a.group / C::ROWS + s);
    }
    int first, n, length;
    const bool ok = seq_rows(a.batch, s, first, n) & seq_length(a.batch, s, pl.page_shift, length);
    if (!ok || (length > 0 && length < n)) {
        if (tid == 0) atomicOr(a.status, kStatusLength);
        length = 0;
    }
    const int64_t all_rows = int64_t(n) * a.group;
    const int tiles = int((all_rows + C::ROWS - 1) / C::ROWS);
    if (nth < 0 || nth >= tiles || n <= args.few_rows / a.group) return;
    const int row0 = (tiles - 1 - nth) * C::ROWS;  // the longest rows first
    const int rows = int(min(int64_t(C::ROWS), all_rows - row0)), pos0 = length - n;
    const int token_lo = row0 / a.group, token_hi = (row0 + rows - 1) / a.group;
    const int any_hi = a.causal ? min(length, pos0 + token_hi + 1) : length;
    const int any_lo = a.window > 0 ? max(0, pos0 + token_lo - a.window + 1) : 0;
    const int j0 = any_lo / BN, steps = max(0, (max(any_hi, 0) + BN - 1) / BN - j0);

    extern __shared__ uint8_t smem_raw[];
    uint8_t *base = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    uint8_t *sm_q = base, *sm_k = sm_q + NQ * C::Q_BYTES, *sm_v = sm_k + 2 * C::KV_BYTES;
    float4 *sm_scale = reinterpret_cast<float4 *>(sm_v + 2 * C::KV_BYTES);  // [2][CHUNKS]: sk, log2 sv, 1/sv
    uint64_t *bars = reinterpret_cast<uint64_t *>(sm_scale + 2 * C::CHUNKS);
    uint64_t *k_full = bars, *k_empty = bars + 2, *v_full = bars + 4, *v_empty = bars + 6, *s_full = bars + 8, *p_full = bars + 10,
             *pv_done = bars + 12, *p_early = bars + 14, *q_full = bars + 16, *o_full = bars + 17;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 19);
    int *err = reinterpret_cast<int *>(tmem_slot + 1);

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full + i, 4);
            mbar_init(v_full + i, 4);
            mbar_init(k_empty + i, 1);
            mbar_init(v_empty + i, 1);
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, 4);
            mbar_init(p_early + i, 4);
            mbar_init(pv_done + i, 1);
            mbar_init(o_full + i, 1);
        }
        mbar_init(q_full, 4 * NQ);
        *err = 0;
        fence_barrier_init();
    }
    if (warp == 0) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

    if (wg < NQ) {
        // ---- softmax: one thread per row
        if constexpr (C::REGS) regs_inc<184>();
        const int r = tid & 127, row = row0 + wg * 128 + r;
        const bool live = wg * 128 + r < rows;
        const int token = live ? row / a.group : 0, head = live ? row - token * a.group : 0;
        const uint32_t lane_base = tmem + (uint32_t((warp & 3) * 32) << 16);
        const uint32_t o_col = lane_base + C::O_COL + wg * D;
        float qs = a.scale * kLog2e;
        {
            // the warp's 32 query rows as f16 in the tile, D / 8 lanes to a row; bf16 rows are brought to
            // [1, 2) by a power of two
            constexpr int LANES = D / 8, PASS = 32 / LANES;  // rows of one load
            const int64_t mine = int64_t(first + token) * a.q_token + int64_t(h * a.group + head) * a.q_head;
            const int alive = __popc(__ballot_sync(0xffffffffu, live));
            const int c = lane % LANES;
            uint8_t *tile = sm_q + wg * C::Q_BYTES + (c / 8) * (128 * 128);
#pragma unroll 8
            for (int i = 0; i < 32; i += PASS) {
                const int from = i + lane / LANES, rr = (warp & 3) * 32 + from;
                const int64_t at = __shfl_sync(0xffffffffu, mine, from);
                Vec<T, 8> x{};
                if (from < alive) x = *reinterpret_cast<const Vec<T, 8> *>(static_cast<const T *>(a.q) + at + c * 8);
                float f[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) f[k] = to_f32(x.v[k]);
                if constexpr (!std::is_same<T, __half>::value) {
                    float m = 0.f;
#pragma unroll
                    for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(f[k]));
#pragma unroll
                    for (int o = LANES / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                    const int e = min(max(int(__float_as_uint(m) >> 23), 1), 253);
                    const float down = __uint_as_float(uint32_t(254 - e) << 23);
#pragma unroll
                    for (int k = 0; k < 8; ++k) f[k] *= down;
                    const int my_e = __shfl_sync(0xffffffffu, e, (lane - i) * LANES & 31);
                    if (lane >= i && lane < i + PASS) qs *= __uint_as_float(uint32_t(my_e) << 23);
                }
                *reinterpret_cast<uint4 *>(tile + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) =
                    make_uint4(pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]), pack_f16x2(f[4], f[5]), pack_f16x2(f[6], f[7]));
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        // keys that this row sees, [lo, hi); a row past the end sees everything and is not written
        const int hi = !live ? 0x7fffffff : a.causal ? min(length, pos0 + token + 1) : length;
        const int lo = live && a.window > 0 ? max(0, pos0 + token - a.window + 1) : 0;
        const int warp_hi = __reduce_min_sync(0xffffffffu, hi), warp_lo = __reduce_max_sync(0xffffffffu, lo);
        float m = ninf, l = 0.f;
        bool good = true;
        for (int j = 0; j < steps && good; ++j) {
            const int st = j & 1, sb = SB == 2 ? st : wg;
            const uint32_t s_col = lane_base + sb * BN;
            good = wait_phase(s_full + sb, SB == 2 ? (j >> 1) & 1 : j & 1, err, kErrWaitFull) &&
                   wait_phase(v_full + st, (j >> 1) & 1, err, kErrWaitFull);  // the scales come with V
            good = __all_sync(0xffffffffu, good);
            if (!good) break;
            tc_fence_after();
            uint32_t x[BN];
#pragma unroll
            for (int c = 0; c < BN; c += 32) tmem_ld32(s_col + c, *reinterpret_cast<uint32_t(*)[32]>(&x[c]));
            tmem_wait_ld();
            const float4 *scales = sm_scale + st * C::CHUNKS;
            const int key0 = (j0 + j) * BN;
            const bool whole = key0 + BN <= warp_hi && key0 >= warp_lo;
            float top = ninf;
            if (whole) {
#pragma unroll
                for (int c = 0; c < BN; c += 16) {
                    float t = fmaxf(__uint_as_float(x[c]), __uint_as_float(x[c + 1]));
#pragma unroll
                    for (int i = 2; i < 16; i += 2) t = max3(t, __uint_as_float(x[c + i]), __uint_as_float(x[c + i + 1]));
                    const float4 sc = scales[c / 16];
                    top = fmaxf(top, fmaf(t, qs * sc.x, sc.y));
                }
            } else {
#pragma unroll
                for (int c = 0; c < BN; c += 16) {
                    const float4 sc = scales[c / 16];
                    const float f0 = qs * sc.x;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int key = key0 + c + i;
                        const float z = key >= lo && key < hi ? fmaf(__uint_as_float(x[c + i]), f0, sc.y) : ninf;
                        x[c + i] = __float_as_uint(z);
                        top = fmaxf(top, z);
                    }
                }
            }
            const bool raise = top > m + kFewStep;
            if (__any_sync(0xffffffffu, raise)) {
                const float to = raise ? top : m;
                if (j > 0) {
                    const float fix = raise ? (m == ninf ? 0.f : ex2(m - to)) : 1.f;
                    l *= fix;
                    good = __all_sync(0xffffffffu, wait_phase(pv_done + wg, (j - 1) & 1, err, kErrWaitDone));
                    if (!good) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) {
                        uint32_t o[16];
                        tmem_ld16(o_col + c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fix);
                        tmem_st16(o_col + c, o);
                    }
                }
                m = to;
            }
            const float off = m == ninf ? 0.f : kFewOffset - m;
            // One of eight pairs takes the polynomial, which relieves the MUFU (16 a clock for the SM, as long
            // as both products of a tile). None / one / two / three of eight, in turns on one GPU, us: 8192-token prompt
            // 617 / 591 / 611 / 618, three chunks of up to 2048 tokens 656 / 614 / 635 / 646, prompt of 1759 49.5 / 47.2 /
            // 48.8 / 49.2, head dim 64 524 / 512 / 523 / 505, head dim 256 351 / 357 / 361 / 360. Masked tiles need 2^-inf = 0.
            auto weights = [&](auto polynomial) {
#pragma unroll
                for (int c = 0; c < BN; c += 32) {
                    uint32_t p[16];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float4 sc = scales[c / 16 + half];
                        const float f0 = decltype(polynomial)::value ? qs * sc.x : 1.f, f1 = decltype(polynomial)::value ? sc.y + off : off;
                        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            float2 z = make_float2(__uint_as_float(x[c + half * 16 + i]), __uint_as_float(x[c + half * 16 + i + 1]));
                            z = ffma2(z, make_float2(f0, f0), make_float2(f1, f1));
                            const float2 e = decltype(polynomial)::value && i == 14 ? ex2_poly(z) : make_float2(ex2(z.x), ex2(z.y));
                            sum = i == 0 ? e : fadd2(sum, e);
                            p[half * 8 + i / 2] = pack_f16x2(e.x, e.y);
                        }
                        l = fmaf(sum.x + sum.y, sc.z, l);
                    }
                    tmem_st16(s_col + c / 2, p);
                    if (c + 32 == C::EARLY) {  // the product may begin on these keys
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(p_early + sb);
                    }
                }
            };
            if (whole)
                weights(std::true_type{});
            else
                weights(std::false_type{});
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + sb);
        }
        if (steps > 0 && good) good = __all_sync(0xffffffffu, wait_phase(o_full + wg, 0, err, kErrWaitDone));
        tc_fence_after();
        const float norm = l == 0.f || !good ? 0.f : 1.f / l;
        T *out = static_cast<T *>(a.out) + int64_t(first + token) * a.o_token + int64_t(h * a.group + head) * a.o_head;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            if (steps > 0) {
                tmem_ld32(o_col + c, o);
                tmem_wait_ld();
            }
            if (!live) continue;
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
                Vec<T, 8> y;
#pragma unroll
                for (int k = 0; k < 8; ++k) y.v[k] = from_f32<T>(norm == 0.f ? 0.f : __uint_as_float(o[i + k]) * norm);
                *reinterpret_cast<Vec<T, 8> *>(out + c + i) = y;
            }
        }
        if (a.lse && live)
            a.lse[int64_t(first + token) * (pl.heads * a.group) + h * a.group + head] =
                l == 0.f ? ninf : (m - kFewOffset + lg2(l)) * 0.6931471805599453f;
    } else if (wg < NQ + C::CONV) {
        // ---- converters: warp w fills keys [w BN / 4, (w + 1) BN / 4) of every tile
        if constexpr (C::REGS) regs_dec<96>();
        constexpr int KEYS = BN / 4, GROUPS = KEYS / 8, RUNS = KEYS / 16;
        const int w = warp & 3;
        const int32_t *table = a.batch.tables + int64_t(s) * a.batch.width;
        uint4 kr[GROUPS * KB];
        // lane: key lane / 4 of a group of eight, 16 channels lane % 4 of a block of 64
        auto key_of = [&](int j, int i) { return (j0 + j) * BN + w * KEYS + i * 16; };
        auto needed = [&](int j, int i) { return j < steps && key_of(j, i) < any_hi && key_of(j, i) + 16 > any_lo; };
        auto pages_of = [&](int j, int (&page)[RUNS]) {
#pragma unroll
            for (int i = 0; i < RUNS; ++i) page[i] = needed(j, i) ? table[key_of(j, i) >> pl.page_shift] : -1;
        };
        auto load = [&](int j, const int (&page)[RUNS], const int8_t *codes, uint4 (&r)[GROUPS * KB]) {
#pragma unroll
            for (int i = 0; i < RUNS; ++i) {
                const bool have = unsigned(page[i]) < unsigned(pl.pages);
                if (!have && lane == 0 && needed(j, i)) atomicOr(a.status, kStatusPage);
                const int key = key_of(j, i);
                const int64_t at = ((int64_t(have ? page[i] : 0) * pl.heads + h) * pl.page_tokens + (key & (pl.page_tokens - 1))) * D;
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int b = 0; b < KB; ++b) {
                        uint4 v = make_uint4(0u, 0u, 0u, 0u);
                        if (have) v = __ldg(reinterpret_cast<const uint4 *>(codes + at + (g * 8 + lane / 4) * D + b * 64 + (lane & 3) * 16));
                        r[(i * 2 + g) * KB + b] = v;
                    }
            }
        };
        auto store = [&](uint8_t *tile, const uint4 (&r)[GROUPS * KB]) {
#pragma unroll
            for (int g = 0; g < GROUPS; ++g)
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    const int row = w * KEYS + g * 8 + lane / 4, c = (lane & 3) * 2;
                    uint8_t *dst = tile + b * (BN * 128) + row * 128;
                    const uint4 v = r[g * KB + b];
                    const uint32_t u[4] = {v.x ^ 0x80808080u, v.y ^ 0x80808080u, v.z ^ 0x80808080u, v.w ^ 0x80808080u};
                    *reinterpret_cast<uint4 *>(dst + ((c ^ (row & 7)) << 4)) =
                        make_uint4(codes_f16x2<0>(u[0]), codes_f16x2<1>(u[0]), codes_f16x2<0>(u[1]), codes_f16x2<1>(u[1]));
                    *reinterpret_cast<uint4 *>(dst + (((c + 1) ^ (row & 7)) << 4)) =
                        make_uint4(codes_f16x2<0>(u[2]), codes_f16x2<1>(u[2]), codes_f16x2<0>(u[3]), codes_f16x2<1>(u[3]));
                }
        };
        // the scales of run `lane` of a tile: loaded a tile ahead, as the page ids are two ahead. Keys without a page
        // (whose codes are zeros) weigh nothing: log2 sv = -inf and 1 / sv = 0
        constexpr float kNoPage = -1.f;
        float2 sc = make_float2(0.f, kNoPage);
        auto load_scales = [&](const int (&page)[RUNS]) {
            sc = make_float2(0.f, kNoPage);
            if (lane >= RUNS) return;
            int pg = page[0];
#pragma unroll
            for (int i = 1; i < RUNS; ++i)
                if (lane == i) pg = page[i];
            if (unsigned(pg) >= unsigned(pl.pages)) return;
            const int64_t ph = int64_t(pg) * pl.heads + h;
            sc = make_float2(sound_scale(pl.k_scale[ph]), sound_scale(pl.v_scale[ph]));
        };
        auto fill = [&](bool v, int j, uint4 (&r)[GROUPS * KB]) {  // wait for the stage, convert, hand over
            const int st = j & 1;
            if (v) {
                const bool zero = zero_block(sc.y);
                const unsigned runs = __ballot_sync(0xffffffffu, zero && lane < RUNS);
#pragma unroll
                for (int i = 0; i < RUNS; ++i)
                    if (runs >> i & 1) {
#pragma unroll
                        for (int k = 0; k < 2 * KB; ++k) r[i * 2 * KB + k] = make_uint4(0u, 0u, 0u, 0u);
                    }
                if (zero) sc.y = kZeroScale;
            }
            if (j >= 2 && !__all_sync(0xffffffffu, wait_phase((v ? v_empty : k_empty) + st, ((j >> 1) - 1) & 1, err, kErrWaitEmpty))) return false;
            // a NaN value scale reaches the rows that see it through its logarithm
            if (v && lane < RUNS)
                sm_scale[st * C::CHUNKS + w * RUNS + lane] =
                    make_float4(sc.x, sc.y == kNoPage ? ninf : lg2(sc.y), sc.y > 0.f ? inverse_scale(sc.y) : 0.f, 0.f);
            store((v ? sm_v : sm_k) + st * C::KV_BYTES, r);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive((v ? v_full : k_full) + st);
            return true;
        };
        int page[RUNS], next[RUNS];
        pages_of(0, page);
        pages_of(1, next);
        if constexpr (C::CONV == 2) {
            // one warpgroup for K, one for V
            const bool v = wg == NQ + 1;
            const int8_t *codes = v ? pl.v_codes : pl.k_codes;
            load(0, page, codes, kr);
            load_scales(page);
            for (int j = 0; j < steps; ++j) {
                if (!fill(v, j, kr)) break;
                if (j + 1 < steps) {
                    load(j + 1, next, codes, kr);
                    load_scales(next);
                    pages_of(j + 2, next);
                }
            }
        } else {
            uint4 vr[GROUPS * KB];
            load(0, page, pl.k_codes, kr);
            load_scales(page);
            for (int j = 0; j < steps; ++j) {
                load(j, page, pl.v_codes, vr);
#pragma unroll
                for (int i = 0; i < RUNS; ++i) page[i] = next[i];
                pages_of(j + 2, next);
                if (!fill(false, j, kr)) break;
                if (j + 1 < steps) load(j + 1, page, pl.k_codes, kr);
                if (!fill(true, j, vr)) break;
                if (j + 1 < steps) load_scales(page);
            }
        }
    } else {
        // ---- MMA: one warp in step, one lane issues, so that the descriptors stay in uniform
        // registers (issued from a branch on the lane they cost 280 cycles each, not 64); a warp for
        // each row tile, whose products then mix, was a tenth slower
        if constexpr (C::REGS) regs_dec<40>();
        if (warp == 4 * (NQ + C::CONV) && steps > 0) {
            constexpr uint32_t idesc_s = umma_idesc_f16_f32(128, BN), idesc_o = umma_idesc_f16_f32(128, D) | (1u << 16);
            const uint64_t q_desc = umma_desc_sw128(smem_u32(sm_q)), k_desc = umma_desc_sw128(smem_u32(sm_k)),
                           v_desc = umma_desc_sw128_mn(smem_u32(sm_v), BN * 128);
            auto wait = [&](uint64_t *bar, int parity) {
                const bool done = wait_phase(bar, parity, err, kErrWaitFull);
                return bool(__all_sync(0xffffffffu, done));
            };
            auto qk = [&](int j, int q) {
                const int sb = SB == 2 ? (j & 1) : q;
                const uint64_t qd = q_desc + (q * C::Q_BYTES >> 4), kd = k_desc + ((j & 1) * C::KV_BYTES >> 4);
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        umma_f16(tmem + sb * BN, qd + ((k / 4) * (128 * 128) + (k & 3) * 32 >> 4),
                                 kd + ((k / 4) * (BN * 128) + (k & 3) * 32 >> 4), idesc_s, k > 0);
                    umma_commit(s_full + sb);
                    if (q == NQ - 1) umma_commit(k_empty + (j & 1));
                }
                __syncwarp();
            };
            auto pv = [&](int j, int q, int k0, int k1) {  // 16-key steps k0 .. k1 - 1
                const int sb = SB == 2 ? (j & 1) : q;
                const uint64_t vd = v_desc + ((j & 1) * C::KV_BYTES >> 4);
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < BN / 16; ++k)
                        if (k >= k0 && k < k1)
                            umma_f16_ts(tmem + C::O_COL + q * D, tmem + sb * BN + k * 8, vd + (k * 2048 >> 4), idesc_o, j > 0 || k > 0);
                    if (k1 == BN / 16) {
                        umma_commit(pv_done + q);
                        if (q == NQ - 1) umma_commit(v_empty + (j & 1));
                        if (j + 1 == steps) umma_commit(o_full + q);
                    }
                }
                __syncwarp();
            };
            bool good = wait(q_full, 0) && wait(k_full, 0);
            for (int q = 0; q < NQ && good; ++q) qk(0, q);
            for (int j = 0; j < steps && good; ++j) {
                const int st = j & 1, phase = (j >> 1) & 1, next = ((j + 1) >> 1) & 1;
                if (SB == 2 && j + 1 < steps) {
                    if (!(good = wait(k_full + (st ^ 1), next))) break;
                    qk(j + 1, 0);
                }
                for (int q = 0; q < NQ; ++q) {
                    const int sb = SB == 2 ? st : q, turn = SB == 2 ? phase : st;
                    if (!(good = (q > 0 || wait(v_full + st, phase)) && wait(p_early + sb, turn))) break;
                    pv(j, q, 0, C::EARLY / 16);
                    if (SB == 1 && j + 1 < steps && q == 0 && !(good = wait(k_full + (st ^ 1), next))) break;
                    if (!(good = wait(p_full + sb, turn))) break;
                    pv(j, q, C::EARLY / 16, BN / 16);
                    if (SB == 1 && j + 1 < steps) qk(j + 1, q);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tmem_dealloc(tmem, 512);
    if (tid == 0 && *err) atomicOr(a.status, kStatusWait);
}

}  // namespace ffnrm::kv
