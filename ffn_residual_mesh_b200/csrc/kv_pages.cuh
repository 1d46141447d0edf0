// Page bookkeeping of the 8-bit paged cache, on the device: which pages are held follows from the
// tables alone, so there is no allocator state to keep in step with them.
//
// fork: child i becomes parent parents[i]'s sequence with room for extra[i] more tokens (-1: an
// empty sequence). Full pages are shared. A partial last page is kept by the lowest child that
// holds it, unless some child holds it as a full page; every other child gets a copy, so an open
// page is never shared. New pages are the lowest free ids, in child order.
// compact: with U pages held, the k-th held page at or above U moves to the k-th free page below
// U. A moved page never lands on a held one, so the old tables stay readable.
//
// One block handles the tables (64 to 256 sequences of 47 pages: 17 us; 128 sequences over 4096 pages:
// 15 us), then every SM moves pages at 94% of the measured copy rate (700 pages in 4 layers: 119 us).
#pragma once

#include "kv_common.cuh"

namespace ffnrm::kv {

constexpr int kPageThreads = 1024;
constexpr int kInfoUsed = 0, kInfoFree = 1, kInfoMoved = 2, kInfoShort = 3;

struct PageArgs {
    const int32_t *tables, *lengths;  // [seqs][width], [seqs]
    const int32_t *parents, *extra;   // fork: [children]
    int32_t *out_tables;              // [children or seqs][out_width]
    int32_t *out_lengths;             // fork: [children]
    int32_t *info;                    // [4]: pages held, pages free, pages copied or moved, pages short
    int32_t *src, *dst, *count;       // the moves, for move_kernel
    int32_t *owner, *list;            // scratch, [pages] each
    int seqs, width, children, out_width, pages, page_shift;
    int *status;
};

// Exclusive scan of one value per thread over the block; `total` is the sum.
template <typename Int>
__device__ __forceinline__ Int block_scan(Int v, Int &total) {
    __shared__ Int sums[kPageThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Int x = v;
    for (int o = 1; o < 32; o <<= 1) {
        const Int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        Int y = sums[lane];
        for (int o = 1; o < 32; o <<= 1) {
            const Int z = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) y += z;
        }
        sums[lane] = y;
    }
    __syncthreads();
    total = sums[kPageThreads / 32 - 1];
    return x - v + (warp ? sums[warp - 1] : 0);
}

// ORs the status bits of all threads (a barrier).
__device__ __forceinline__ int block_or(int bits, int *shared) {
    if (bits) atomicOr(shared, bits);
    __syncthreads();
    return *shared;
}

// f(row, column, index) for every entry of a [rows][width] table, kPageBatch entries of a thread at a
// time, so that their loads are under way together: get loads, put uses.
constexpr int kPageBatch = 8;
template <typename Index, typename Get, typename Put>
__device__ __forceinline__ void for_entries_of(Index total, Index width, Get get, Put put) {
    for (Index e0 = threadIdx.x; e0 < total; e0 += kPageThreads * kPageBatch) {
        int v[kPageBatch], row[kPageBatch], col[kPageBatch];
#pragma unroll
        for (int i = 0; i < kPageBatch; ++i) {
            const Index e = e0 + i * kPageThreads;
            row[i] = int(e / width);
            col[i] = int(e - Index(row[i]) * width);
            if (e < total) v[i] = get(row[i], col[i], int64_t(e));
        }
#pragma unroll
        for (int i = 0; i < kPageBatch; ++i) {
            const Index e = e0 + i * kPageThreads;
            if (e < total) put(row[i], col[i], int64_t(e), v[i]);
        }
    }
}
template <typename Get, typename Put>
__device__ __forceinline__ void for_entries(int rows, int width, Get get, Put put) {
    const int64_t total = int64_t(rows) * width;
    if (total < (1 << 30))  // 64-bit divisions would take longer than the loads
        for_entries_of<uint32_t>(uint32_t(total), uint32_t(width), get, put);
    else
        for_entries_of<int64_t>(total, width, get, put);
}

// One block. Shared memory: a bit per page, five integers per child. Bound by the latency of the
// dependent loads (parent, length, table entry) and a dozen barriers. lengths, parents and extra are read before the
// first barrier and out_lengths is written behind the last look at the tables, so it may lie on any of them.
__global__ void __launch_bounds__(kPageThreads) fork_kernel(PageArgs a) {
    extern __shared__ uint32_t held[];
    __shared__ int flags;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const int words = (a.pages + 31) / 32, P = 1 << a.page_shift, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int *full = reinterpret_cast<int *>(held + words), *open = full + a.children, *need = open + a.children, *from = need + a.children,
        *grown = from + a.children;
    for (int i = tid; i < words; i += kPageThreads) held[i] = 0;
    if (tid == 0) flags = 0;
    __syncthreads();
    int bad = 0;
    // each child's parent, full pages and open page
    for (int c = tid; c < a.children; c += kPageThreads) {
        const int p = a.parents[c], more = a.extra[c];
        int length = 0, parent = -1;
        if (p >= 0 && p < a.seqs) {
            length = a.lengths[p];
            if (length >= 0 && length <= (int64_t(a.width) << a.page_shift) && length <= (int64_t(a.out_width) << a.page_shift))
                parent = p;
            else {
                length = 0;
                bad |= kStatusLength;
            }
        } else if (p != -1) {
            bad |= kStatusLength;
        }
        const int nf = length >> a.page_shift;
        int op = -1;
        if (parent >= 0 && (length & (P - 1))) {
            op = a.tables[int64_t(parent) * a.width + nf];
            if (op < 0 || op >= a.pages) {
                bad |= kStatusPage;
                op = -1;
            }
        }
        if (op >= 0) a.owner[op] = 0x7fffffff;
        int grow = more;
        if (more < 0 || int64_t(length) + more > (int64_t(a.out_width) << a.page_shift)) {
            bad |= kStatusLength;
            grow = 0;
        }
        from[c] = parent;
        full[c] = nf;
        open[c] = op;
        need[c] = ((length + grow + P - 1) >> a.page_shift) - nf;
        grown[c] = length + grow;
    }
    block_or(bad, &flags);
    // shared pages: a warp per child
    for (int c = warp; c < a.children; c += kPageThreads / 32) {
        const int nf = full[c];
        const int32_t *row = a.tables + int64_t(max(0, from[c])) * a.width;
        int32_t *out = a.out_tables + int64_t(c) * a.out_width;
#pragma unroll 4
        for (int w = lane; w < nf; w += 32) {
            int id = row[w];
            if (id >= 0 && id < a.pages) {
                atomicOr(&held[id >> 5], 1u << (id & 31));
            } else {
                bad |= kStatusPage;
                id = -1;
            }
            out[w] = id;
        }
    }
    for (int c = tid; c < a.children; c += kPageThreads)
        if (open[c] >= 0) atomicMin(&a.owner[open[c]], c);
    bad = block_or(bad, &flags);
    // who keeps an open page; decided before any of them is marked
    for (int c = tid; c < a.children; c += kPageThreads) {
        const int op = open[c];
        if (op < 0) continue;
        const bool keep = __ldcg(&a.owner[op]) == c && !((held[op >> 5] >> (op & 31)) & 1);
        if (keep) {
            need[c] -= 1;
            full[c] |= int(0x80000000);  // the open page is kept
        }
    }
    __syncthreads();
    for (int c = tid; c < a.children; c += kPageThreads)
        if (open[c] >= 0 && full[c] < 0) atomicOr(&held[open[c] >> 5], 1u << (open[c] & 31));
    __syncthreads();
    // free pages in ascending order
    const int per = (words + kPageThreads - 1) / kPageThreads, w0 = tid * per, w1 = min(words, w0 + per);
    auto free_bits = [&](int w) {
        const int n = a.pages - w * 32;
        return ~held[w] & (n >= 32 ? 0xffffffffu : (1u << n) - 1u);
    };
    int mine = 0, free_total;
    int64_t want = 0, want_total;  // 4096 children may ask for 2^26 pages each
    for (int w = w0; w < w1; ++w) mine += __popc(free_bits(w));
    int rank = block_scan(mine, free_total);
    const int cper = (a.children + kPageThreads - 1) / kPageThreads, c0 = tid * cper, c1 = min(a.children, c0 + cper);
    int copies = 0, copies_total;
    for (int c = c0; c < c1; ++c) {
        want += need[c];
        copies += open[c] >= 0 && full[c] >= 0;
    }
    int64_t offset = block_scan(want, want_total);
    int copy_at = block_scan(copies, copies_total);
    const int shortage = int(min(max(want_total - free_total, int64_t(0)), int64_t(0x7fffffff)));
    const bool refuse = shortage || bad;
    for (int w = w0; w < w1 && rank < want_total; ++w) {
        for (uint32_t b = free_bits(w); b; b &= b - 1) {
            if (rank < want_total) a.list[rank] = w * 32 + __ffs(b) - 1;
            ++rank;
        }
    }
    __syncthreads();
    int *count = from;  // from here on: a child's new pages
    for (int c = c0; c < c1; ++c) {
        const int n = need[c];
        if (open[c] >= 0 && full[c] >= 0 && !refuse) {
            a.src[copy_at] = open[c];
            a.dst[copy_at] = a.list[offset];
            ++copy_at;
        }
        need[c] = refuse ? 0 : int(offset);
        count[c] = n;
        offset += n;
        a.out_lengths[c] = refuse ? 0 : grown[c];
    }
    if (tid == 0) {
        a.info[kInfoUsed] = a.pages - free_total + (refuse ? 0 : int(want_total));
        a.info[kInfoFree] = free_total - (refuse ? 0 : int(want_total));
        a.info[kInfoMoved] = refuse ? 0 : copies_total;
        a.info[kInfoShort] = shortage;
        *a.count = refuse ? 0 : copies_total;
        if (refuse) atomicOr(a.status, bad | (shortage ? kStatusPages : 0));
    }
    __syncthreads();
    // the rest of each row: the open page or its copy, new pages, none
    for (int c = warp; c < a.children; c += kPageThreads / 32) {
        const bool keep = full[c] < 0;
        const int nf = full[c] & 0x7fffffff, first = nf + (keep ? 1 : 0), n = count[c], at = need[c];
        int32_t *out = a.out_tables + int64_t(c) * a.out_width;
#pragma unroll 4
        for (int w = refuse ? lane : nf + lane; w < a.out_width; w += 32) {
            const int i = w - first;
            const int fresh = __ldcg(a.list + max(0, min(at + i, a.pages - 1)));
            out[w] = refuse ? -1 : i < 0 ? open[c] : i < n ? fresh : -1;
        }
    }
}

// One block. Shared memory: a bit per page, an integer per sequence.
__global__ void __launch_bounds__(kPageThreads) compact_kernel(PageArgs a) {
    extern __shared__ uint32_t held[];
    __shared__ int flags;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const int words = (a.pages + 31) / 32, P = 1 << a.page_shift, tid = threadIdx.x;
    for (int i = tid; i < words; i += kPageThreads) held[i] = 0;
    if (tid == 0) flags = 0;
    __syncthreads();
    int bad = 0;
    // pages of each sequence; 0 for a length that its row cannot hold
    int *full = reinterpret_cast<int *>(held + words);
    for (int s = tid; s < a.seqs; s += kPageThreads) {
        const int length = a.lengths[s];
        const bool fits = length >= 0 && length <= (int64_t(a.width) << a.page_shift);
        full[s] = fits ? (length + P - 1) >> a.page_shift : 0;
        if (!fits) bad |= kStatusLength;
    }
    __syncthreads();
    for_entries(
        a.seqs, a.width, [&](int, int, int64_t e) { return a.tables[e]; },
        [&](int s, int w, int64_t, int id) {
            if (w >= full[s]) return;
            if (id >= 0 && id < a.pages)
                atomicOr(&held[id >> 5], 1u << (id & 31));
            else
                bad |= kStatusPage;
        });
    bad = block_or(bad, &flags);
    const int per = (words + kPageThreads - 1) / kPageThreads, w0 = tid * per, w1 = min(words, w0 + per);
    int mine = 0, used;
    for (int w = w0; w < w1; ++w) mine += __popc(held[w]);
    int before = block_scan(mine, used);  // held pages below this thread's words
    // holes below `used`, in order
    for (int w = w0; w < w1; ++w) {
        const int inside = used - w * 32;
        if (inside <= 0) break;
        uint32_t b = ~held[w] & (inside >= 32 ? 0xffffffffu : (1u << inside) - 1u);
        int rank = w * 32 - before;
        before += __popc(held[w]);
        for (; b; b &= b - 1) a.list[rank++] = w * 32 + __ffs(b) - 1;
    }
    __syncthreads();
    // the held pages at or above `used`, in order
    int high = 0, high_total;
    for (int w = w0; w < w1; ++w) {
        const int inside = used - w * 32;
        const uint32_t lowmask = inside <= 0 ? 0u : inside >= 32 ? 0xffffffffu : (1u << inside) - 1u;
        high += __popc(held[w] & ~lowmask);
    }
    int rank = block_scan(high, high_total);
    for (int w = w0; w < w1; ++w) {
        const int inside = used - w * 32;
        const uint32_t lowmask = inside <= 0 ? 0u : inside >= 32 ? 0xffffffffu : (1u << inside) - 1u;
        for (uint32_t b = held[w] & ~lowmask; b; b &= b - 1) a.src[rank++] = w * 32 + __ffs(b) - 1;
    }
    __syncthreads();
    // the k-th held page above goes to the k-th hole below
    for (int k = tid; k < high_total; k += kPageThreads) {
        const int to = __ldcg(a.list + k);
        a.owner[__ldcg(a.src + k)] = to;
        a.dst[k] = to;
    }
    if (tid == 0) {
        a.info[kInfoUsed] = used;
        a.info[kInfoFree] = a.pages - used;
        a.info[kInfoMoved] = bad ? 0 : high_total;
        a.info[kInfoShort] = 0;
        *a.count = bad ? 0 : high_total;
        if (bad) atomicOr(a.status, bad);
    }
    __syncthreads();
    // bad tables: nothing moves and the rows are handed on as they are
    for_entries(
        a.seqs, a.width,
        [&](int, int, int64_t e) { return a.tables[e]; },
        [&](int s, int w, int64_t e, int id) {
            if (!bad) id = w >= full[s] ? -1 : id >= used ? __ldcg(&a.owner[id]) : id;
            a.out_tables[e] = id;
        });
}

struct MoveArgs {
    int8_t *k_codes, *v_codes;   // all layers
    float *k_scale, *v_scale;
    const int32_t *src, *dst, *count;
    int layers, pages, heads, page_bytes;  // page_bytes: codes of one page of one layer
    int most;                              // upper bound of the list; its length without a count
    int *status;
};

constexpr int kMoveChunk = 32768, kMoveLoads = kMoveChunk / 16 / 256;

// Copies every listed page in every layer, kMoveChunk bytes of codes per block step. Bound by reading and
// writing them once: eight 16-byte loads under way per thread, the next step's page ids read ahead.
__global__ void __launch_bounds__(256) move_kernel(MoveArgs a) {
    asm volatile("griddepcontrol.wait;\n" ::: "memory");  // the list is the kernel's before
    const int moves = a.count ? min(*a.count, a.most) : a.most, chunks = (a.page_bytes + kMoveChunk - 1) / kMoveChunk;
    const int per_move = a.layers * 2 * chunks;
    const int64_t items = int64_t(moves) * per_move;
    int64_t i = blockIdx.x;
    if (i >= items) return;
    int m = int(i / per_move);
    int src = a.src[m], dst = a.dst[m];
    while (true) {
        const int part = int(i - int64_t(m) * per_move), chunk = part % chunks, kv = part / chunks & 1, layer = part / chunks >> 1;
        const int64_t next = i + gridDim.x;
        const bool more = next < items;
        const int next_m = more ? int(next / per_move) : m;
        const int next_src = a.src[next_m], next_dst = a.dst[next_m];
        if (unsigned(src) < unsigned(a.pages) && unsigned(dst) < unsigned(a.pages)) {
            const int64_t from = int64_t(layer) * a.pages + src, to = int64_t(layer) * a.pages + dst;
            int8_t *codes = kv ? a.v_codes : a.k_codes;
            const uint4 *x = reinterpret_cast<const uint4 *>(codes + from * a.page_bytes + int64_t(chunk) * kMoveChunk);
            uint4 *y = reinterpret_cast<uint4 *>(codes + to * a.page_bytes + int64_t(chunk) * kMoveChunk);
            const int n = min(kMoveChunk, a.page_bytes - chunk * kMoveChunk) / 16;
            uint4 v[kMoveLoads];
#pragma unroll
            for (int j = 0; j < kMoveLoads; ++j)
                if (int(threadIdx.x) + j * 256 < n) v[j] = x[threadIdx.x + j * 256];
#pragma unroll
            for (int j = 0; j < kMoveLoads; ++j)
                if (int(threadIdx.x) + j * 256 < n) y[threadIdx.x + j * 256] = v[j];
            if (chunk == 0) {
                float *scale = kv ? a.v_scale : a.k_scale;
                for (int h = threadIdx.x; h < a.heads; h += 256) scale[to * a.heads + h] = scale[from * a.heads + h];
            }
        } else if (threadIdx.x == 0) {
            atomicOr(a.status, kStatusPage);
        }
        if (!more) return;
        i = next, m = next_m, src = next_src, dst = next_dst;
    }
}

}  // namespace ffnrm::kv
