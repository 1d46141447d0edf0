// C ABI of the 8-bit paged cache and its operators (include/ffnrm.h, ffnrm_rotary, ffnrm_kv_*).
#include "ffnrm.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <mutex>
#include <new>

#include "kv_append.cuh"
#include "kv_attend_many.cuh"
#include "kv_common.cuh"
#include "kv_pages.cuh"
#include "kv_rotary.cuh"

namespace ffnrm {
int set_error(int code, const char *message);  // ffnrm.cu
}

namespace {

using namespace ffnrm::kv;

int fail(int code, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return ffnrm::set_error(code, buf);
}

#define KV_CUDA(expr)                                                                                        \
    do {                                                                                                     \
        cudaError_t _e = (expr);                                                                             \
        if (_e != cudaSuccess)                                                                               \
            return fail(FFNRM_ERR_CUDA, "%s failed at %s:%d: %s", #expr, __FILE__, __LINE__, cudaGetErrorString(_e)); \
    } while (0)

struct DeviceGuard {
    int prev = -1;
    explicit DeviceGuard(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev != dev) cudaSetDevice(dev);
    }
    ~DeviceGuard() {
        int cur = -1;
        if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
    }
};

bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
// Whether two ranges of memory share a byte.
bool share_bytes(const void *a, size_t na, const void *b, size_t nb) {
    const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return na && nb && x < y + nb && y < x + na;
}
size_t type_size(int dtype) { return dtype == FFNRM_F32 ? 4 : 2; }

// Whether a row block can be read in 16-byte accesses (a single token's or head's stride is never used).
bool wide(const ffnrm_rows &r, int dtype, int tokens, int heads) {
    const int64_t n = 16 / int64_t(type_size(dtype));
    return aligned(r.data, 16) && (tokens == 1 || r.token_stride % n == 0) && (heads == 1 || r.head_stride % n == 0);
}

int check_rows(const char *name, const ffnrm_rows *r, int dtype) {
    if (!r || !r->data) return fail(FFNRM_ERR_ARG, "%s: null rows", name);
    if (!aligned(r->data, type_size(dtype))) return fail(FFNRM_ERR_ARG, "%s: misaligned rows", name);
    return FFNRM_OK;
}

// The least |e + a stride| over whole numbers |a| <= most is below dim.
bool comes_near(int64_t e, int64_t stride, int64_t most, int64_t dim) {
    if (stride == 0 || most <= 0) return std::abs(e) < dim;
    const int64_t a = -e / stride;  // the nearest is one of its neighbours, or the end of the range
    for (int64_t i = a - 1; i <= a + 1; ++i)
        if (std::abs(e + std::clamp(i, -most, most) * stride) < dim) return true;
    return false;
}

// Row blocks of `tokens` rows: x with hx heads and y with hy, rows of dim elements of one type.
struct RowPair {
    int64_t tokens, hx, hy, dim;
    size_t size;
};
// First byte and end of a block.
void extent(const ffnrm_rows &r, int64_t tokens, int64_t heads, const RowPair &p, uintptr_t &lo, uintptr_t &hi) {
    const int64_t t = (tokens - 1) * r.token_stride, h = (heads - 1) * r.head_stride;
    lo = reinterpret_cast<uintptr_t>(r.data) + (std::min<int64_t>(t, 0) + std::min<int64_t>(h, 0)) * int64_t(p.size);
    hi = reinterpret_cast<uintptr_t>(r.data) + (std::max<int64_t>(t, 0) + std::max<int64_t>(h, 0) + p.dim) * int64_t(p.size);
}
bool same_rows(const ffnrm_rows &x, const ffnrm_rows &y, const RowPair &p) {
    return x.data == y.data && p.hx == p.hy && (p.tokens == 1 || x.token_stride == y.token_stride) &&
           (p.hx == 1 || x.head_stride == y.head_stride);
}
// Whether x and y share an element. Blocks that lie in one another's gaps (slices of packed rows) do not, which is
// found where they have one token stride; with two different ones they count as sharing.
bool rows_meet(const ffnrm_rows &x, const ffnrm_rows &y, const RowPair &p) {
    uintptr_t x0, x1, y0, y1;
    extent(x, p.tokens, p.hx, p, x0, x1);
    extent(y, p.tokens, p.hy, p, y0, y1);
    if (x0 >= y1 || y0 >= x1) return false;
    if (p.tokens > 1 && x.token_stride != y.token_stride) return true;
    const int64_t d = (reinterpret_cast<intptr_t>(y.data) - reinterpret_cast<intptr_t>(x.data)) / int64_t(p.size);
    const bool alike = x.head_stride == y.head_stride;  // then only the difference of the heads counts
    for (int64_t i = 0; i < p.hx; ++i)
        for (int64_t j = 0; j < (alike && i ? 1 : p.hy); ++j)
            if (comes_near(d + j * y.head_stride - i * x.head_stride, x.token_stride, p.tokens - 1, p.dim)) return true;
    return false;
}
// Whether two rows of a block share an element.
bool rows_fold(const ffnrm_rows &x, int64_t tokens, int64_t heads, int64_t dim) {
    const int64_t st = x.token_stride, sh = x.head_stride;
    if (sh >= dim && st >= (heads - 1) * sh + dim) return false;  // rows one behind another
    if (tokens > 1 && std::abs(st) < dim) return true;
    for (int64_t b = 1; b < heads; ++b)
        if (comes_near(b * sh, st, tokens - 1, dim)) return true;
    return false;
}
// Rows that a kernel writes: apart from one another, and the rows that it reads meanwhile or apart from them.
int check_written(const char *name, const ffnrm_rows &y, const char *from, const ffnrm_rows &x, const RowPair &p) {
    if (rows_fold(y, p.tokens, p.hy, p.dim)) return fail(FFNRM_ERR_ARG, "%s: rows lie on one another", name);
    if (!same_rows(x, y, p) && rows_meet(x, y, p)) return fail(FFNRM_ERR_ARG, "%s must be %s itself or lie apart from it", name, from);
    return FFNRM_OK;
}

int check_table(const float *table, int rotary_dim, int max_positions, int head_dim, int flags, int allowed) {
    if (!table || !aligned(table, 4)) return fail(FFNRM_ERR_ARG, "null or misaligned rotary table");
    if (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > head_dim)
        return fail(FFNRM_ERR_ARG, "rotary_dim=%d must be even, positive and at most head_dim=%d", rotary_dim, head_dim);
    if (max_positions <= 0) return fail(FFNRM_ERR_ARG, "max_positions=%d must be positive", max_positions);
    if (flags & ~allowed) return fail(FFNRM_ERR_ARG, "unknown rotary flags %d", flags);
    return FFNRM_OK;
}

constexpr int kRotaryHeads = 4;

template <typename T, bool INTERLEAVED, int VEC, int HEADS>
void launch_rotary_t(const RotaryArgs &a, float sign, cudaStream_t st) {
    const int64_t n = int64_t(a.tokens) * ((a.heads + HEADS - 1) / HEADS) * rotary_units<INTERLEAVED, VEC>(a.dim, a.rot);
    rotary_kernel<T, INTERLEAVED, VEC, HEADS><<<unsigned((n + 255) / 256), 256, 0, st>>>(a, sign);
}

template <typename T, bool INTERLEAVED>
void launch_rotary(const RotaryArgs &a, float sign, bool wide_rows, cudaStream_t st) {
    constexpr int N = 16 / int(sizeof(T));
    // few rows: one head to a thread, so that there are threads for every SM
    const bool few = int64_t(a.tokens) * a.heads < 16384;
    if (!wide_rows || !rotary_fits(INTERLEAVED, N, a.dim, a.rot, a.table))
        launch_rotary_t<T, INTERLEAVED, 1, 1>(a, sign, st);
    else if (few)
        launch_rotary_t<T, INTERLEAVED, N, 1>(a, sign, st);
    else
        launch_rotary_t<T, INTERLEAVED, N, kRotaryHeads>(a, sign, st);
}

// What a device needs once: the blocks of each few-rows variant that it holds (by type, head dim and row
// tiles) and the workspace of partials for them.
struct DeviceSetup {
    bool done = false;
    int sms = 0, grid[2][3][2] = {};
    size_t floats[3] = {};
};

}  // namespace

struct ffnrm_kv {
    int device = 0;
    ffnrm_kv_config cfg{};
    int page_shift = 0;
    int8_t *k_codes = nullptr, *v_codes = nullptr;
    float *k_scale = nullptr, *v_scale = nullptr;
    int num_sms = 148;
    const DeviceSetup *setup = nullptr;
    int *status = nullptr;       // what kernels could not use, kStatus* bits
    float *partial = nullptr;    // pieces of attention items cut between blocks
    int *counters = nullptr;     // their arrivals, zero between calls
    void *scratch = nullptr;     // the handle's memory: all of the above and the page lists of fork / compact
    int32_t *src = nullptr, *dst = nullptr, *owner = nullptr, *list = nullptr, *count = nullptr;
};

namespace {

int check_kv(ffnrm_kv *kv, int layer) {
    if (!kv) return fail(FFNRM_ERR_ARG, "null cache");
    if (layer < 0 || layer >= kv->cfg.n_layers)
        return fail(FFNRM_ERR_ARG, "layer %d out of range [0, %d)", layer, kv->cfg.n_layers);
    return FFNRM_OK;
}

int check_batch(ffnrm_kv *kv, const ffnrm_kv_batch *b) {
    if (!b) return fail(FFNRM_ERR_ARG, "null batch");
    if (b->seqs < 0 || b->seqs > kv->cfg.max_seqs)
        return fail(FFNRM_ERR_ARG, "seqs=%d outside [0, max_seqs=%d]", b->seqs, kv->cfg.max_seqs);
    if (b->rows < 0 || b->table_width < 0) return fail(FFNRM_ERR_ARG, "rows and table_width must not be negative");
    if ((int64_t(b->table_width) << kv->page_shift) > (int64_t(1) << 30))
        return fail(FFNRM_ERR_ARG, "table_width=%d addresses more than 2^30 tokens", b->table_width);
    if (!b->starts && b->rows != b->seqs)
        return fail(FFNRM_ERR_ARG, "without starts there is one row per sequence: rows=%d, seqs=%d", b->rows, b->seqs);
    if (b->seqs > 0 && (!b->lengths || (b->table_width > 0 && !b->tables)))
        return fail(FFNRM_ERR_ARG, "null tables or lengths");
    if (!aligned(b->tables, 4) || !aligned(b->lengths, 4) || !aligned(b->starts, 4))
        return fail(FFNRM_ERR_ARG, "tables, lengths and starts must be 4-byte aligned");
    return FFNRM_OK;
}

Pool layer_pool(const ffnrm_kv *kv, int layer) {
    const ffnrm_kv_config &c = kv->cfg;
    const int64_t ph = int64_t(layer) * c.n_pages * c.kv_heads, codes = ph * c.page_tokens * c.head_dim;
    return Pool{kv->k_codes + codes, kv->v_codes + codes, kv->k_scale + ph, kv->v_scale + ph,
                c.n_pages,           c.kv_heads,          c.head_dim,       c.page_tokens,    kv->page_shift};
}

Batch batch_view(const ffnrm_kv_batch *b) { return Batch{b->tables, b->lengths, b->starts, b->seqs, b->table_width, b->rows}; }

template <typename T>
void launch_append(const AppendArgs &a, bool vec, bool interleaved, unsigned grid, cudaStream_t st) {
    if (vec && interleaved)
        append_kernel<T, true, true><<<grid, 256, 0, st>>>(a);
    else if (vec)
        append_kernel<T, true, false><<<grid, 256, 0, st>>>(a);
    else if (interleaved)
        append_kernel<T, false, true><<<grid, 256, 0, st>>>(a);
    else
        append_kernel<T, false, false><<<grid, 256, 0, st>>>(a);
}

constexpr int kFewWarps = 8, kFewMinUnits = 1;

// f(kernel, dynamic shared memory, floats of one partial) of the variant for rows of type T,
// head dim D and NT tiles of eight rows.
template <typename F>
int with_few(int dtype, int dim, int nt, F f) {
#define FEW(T, D, NT) return f(attend_few_kernel<T, D, NT, kFewWarps>, few_smem<D, NT, kFewWarps>(), few_slot<D, NT>())
#define FEW_T(T)                                                                                              \
    switch (dim * 4 + nt) {                                                                                   \
        case 64 * 4 + 1: FEW(T, 64, 1);                                                                       \
        case 64 * 4 + 2: FEW(T, 64, 2);                                                                       \
        case 128 * 4 + 1: FEW(T, 128, 1);                                                                     \
        case 128 * 4 + 2: FEW(T, 128, 2);                                                                     \
        case 256 * 4 + 1: FEW(T, 256, 1);                                                                     \
        default: FEW(T, 256, 2);                                                                              \
    }
    if (dtype == FFNRM_F16) {
        FEW_T(__half)
    } else {
        FEW_T(__nv_bfloat16)
    }
#undef FEW_T
#undef FEW
}

int dim_index(int dim) { return dim == 64 ? 0 : dim == 128 ? 1 : 2; }

template <typename T>
cudaError_t prepare_many() {
    cudaError_t e = cudaFuncSetAttribute(attend_many_kernel<T, 64>, cudaFuncAttributeMaxDynamicSharedMemorySize, Many<64>::SMEM);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(attend_many_kernel<T, 128>, cudaFuncAttributeMaxDynamicSharedMemorySize, Many<128>::SMEM);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(attend_many_kernel<T, 256>, cudaFuncAttributeMaxDynamicSharedMemorySize, Many<256>::SMEM);
    return e;
}

int device_setup(int device, const DeviceSetup *&out) {
    static std::mutex lock;
    static DeviceSetup table[64];
    if (device >= 64) return fail(FFNRM_ERR_ARG, "device %d beyond the supported 64", device);
    const std::lock_guard<std::mutex> hold(lock);
    DeviceSetup &d = table[device];
    out = &d;
    if (d.done) return FFNRM_OK;
    KV_CUDA(cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, device));
    for (int dtype : {FFNRM_F16, FFNRM_BF16})
        for (int dim : {64, 128, 256})
            for (int nt : {1, 2}) {
                const int rc = with_few(dtype, dim, nt, [&](auto kernel, int smem, int slot) {
                    int per_sm = 0;
                    KV_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
                    KV_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kFewWarps * 32, smem));
                    const int i = dim_index(dim), grid = std::max(1, per_sm) * d.sms;
                    d.grid[dtype][i][nt - 1] = grid;
                    d.floats[i] = std::max(d.floats[i], size_t(2) * grid * slot);
                    return int(FFNRM_OK);
                });
                if (rc) return rc;
            }
    KV_CUDA(prepare_many<__half>());
    KV_CUDA(prepare_many<__nv_bfloat16>());
    // a bit for each of up to 2^20 pages, and 20 or 4 bytes for each of up to 4096 sequences
    KV_CUDA(cudaFuncSetAttribute(fork_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (1 << 17) + 20 * 4096));
    KV_CUDA(cudaFuncSetAttribute(compact_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (1 << 17) + 4 * 4096));
    d.done = true;
    return FFNRM_OK;
}

// Sequences with more query rows (tokens x group) than this take the tcgen05 kernel. It has one block for 256
// rows of a kv head over all keys, the few-rows kernel splits the keys: where the blocks fill the GPU
// the first is as fast from 64 rows on (16 sequences of up to 128 tokens x 8: 109 us, 146 with 256
// here), where they do not the second up to 256 (2 sequences of up to 32 x 8 over 16k keys: 194 us, 281).
int few_rows(const ffnrm_kv *kv, const ffnrm_kv_batch *batch, int group) {
    return int64_t(batch->rows) * group * kv->cfg.kv_heads < int64_t(256) * kv->num_sms ? 256 : 64;
}

int launch_few(ffnrm_kv *kv, const AttendArgs &a, int dtype, int most_rows, cudaStream_t st) {
    // rows of one kv head that a sequence brings on average
    const int64_t rows = int64_t(a.group) * ((a.batch.rows + a.batch.seqs - 1) / a.batch.seqs);
    const int nt = rows > 8 ? 2 : 1;
    const FewArgs f{a, kv->partial, kv->counters, kFewMinUnits, most_rows};
    return with_few(dtype, kv->cfg.head_dim, nt, [&](auto kernel, int smem, int) {
        kernel<<<unsigned(kv->setup->grid[dtype][dim_index(kv->cfg.head_dim)][nt - 1]), kFewWarps * 32, smem, st>>>(f);
        KV_CUDA(cudaGetLastError());
        return int(FFNRM_OK);
    });
}

template <typename T, int D>
int launch_many_t(ffnrm_kv *kv, const ManyArgs &m, cudaStream_t st) {
    attend_many_kernel<T, D><<<unsigned(m.slots) * unsigned(kv->cfg.kv_heads), Many<D>::THREADS, Many<D>::SMEM, st>>>(m);
    KV_CUDA(cudaGetLastError());
    return FFNRM_OK;
}

int launch_many(ffnrm_kv *kv, const AttendArgs &a, int dtype, int few_rows, bool alone, cudaStream_t st) {
    const int tile = kv->cfg.head_dim == 256 ? Many<256>::ROWS : Many<128>::ROWS;
    const int64_t slots = many_slots(a.batch.seqs, a.batch.rows, a.group, tile);
    if (slots * kv->cfg.kv_heads > 0x7fffffff) return fail(FFNRM_ERR_ARG, "rows=%d are too many for one call", a.batch.rows);
    const ManyArgs m{a, int(slots), few_rows, alone};
    const bool f16 = dtype == FFNRM_F16;
    if (kv->cfg.head_dim == 64) return f16 ? launch_many_t<__half, 64>(kv, m, st) : launch_many_t<__nv_bfloat16, 64>(kv, m, st);
    if (kv->cfg.head_dim == 128) return f16 ? launch_many_t<__half, 128>(kv, m, st) : launch_many_t<__nv_bfloat16, 128>(kv, m, st);
    return f16 ? launch_many_t<__half, 256>(kv, m, st) : launch_many_t<__nv_bfloat16, 256>(kv, m, st);
}

int launch_moves(ffnrm_kv *kv, const int32_t *src, const int32_t *dst, const int32_t *count, int most, cudaStream_t st) {
    const ffnrm_kv_config &c = kv->cfg;
    const int page_bytes = c.kv_heads * c.page_tokens * c.head_dim;
    MoveArgs m{kv->k_codes, kv->v_codes, kv->k_scale, kv->v_scale, src,  dst,       count,
               c.n_layers,  c.n_pages,   c.kv_heads,  page_bytes,  most, kv->status};
    const int64_t items = int64_t(most) * c.n_layers * 2 * ((page_bytes + kMoveChunk - 1) / kMoveChunk);
    const unsigned grid = unsigned(std::min<int64_t>(items, int64_t(kv->num_sms) * 8));
    // behind fork / compact as a dependent launch: it waits for the list itself
    cudaLaunchConfig_t lc{};
    lc.gridDim = dim3(grid);
    lc.blockDim = dim3(256);
    lc.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = &attr;
    lc.numAttrs = count ? 1 : 0;
    KV_CUDA(cudaLaunchKernelEx(&lc, move_kernel, m));
    return FFNRM_OK;
}

}  // namespace

extern "C" {

int ffnrm_rotary(const ffnrm_rows *x, const ffnrm_rows *y, int dtype, int tokens, int heads, int head_dim,
                 const int32_t *positions, const float *table, int rotary_dim, int max_positions, int flags,
                 void *stream) {
    if (dtype < FFNRM_F16 || dtype > FFNRM_F32) return fail(FFNRM_ERR_ARG, "unknown element type %d", dtype);
    if (tokens < 0 || heads < 0 || head_dim <= 0)
        return fail(FFNRM_ERR_ARG, "tokens=%d, heads=%d, head_dim=%d are no shape", tokens, heads, head_dim);
    int rc = check_table(table, rotary_dim, max_positions, head_dim, flags, FFNRM_ROTARY_INTERLEAVED | FFNRM_ROTARY_INVERSE);
    if (rc) return rc;
    if (tokens == 0 || heads == 0) return FFNRM_OK;
    if ((rc = check_rows("x", x, dtype)) || (rc = check_rows("y", y, dtype))) return rc;
    if ((rc = check_written("y", *y, "x", *x, RowPair{tokens, heads, heads, head_dim, type_size(dtype)}))) return rc;
    if (!positions || !aligned(positions, 4)) return fail(FFNRM_ERR_ARG, "null or misaligned positions");
    if (int64_t(tokens) * heads * head_dim / 256 > 0x7fffffff) return fail(FFNRM_ERR_ARG, "tokens=%d are too many for one call", tokens);
    const RotaryArgs a{x->data, y->data, positions, table, x->token_stride, x->head_stride, y->token_stride, y->head_stride,
                       tokens, heads, head_dim, rotary_dim, max_positions};
    const bool vec = wide(*x, dtype, tokens, heads) && wide(*y, dtype, tokens, heads), inter = flags & FFNRM_ROTARY_INTERLEAVED;
    const float sign = flags & FFNRM_ROTARY_INVERSE ? -1.f : 1.f;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == FFNRM_F16)
        inter ? launch_rotary<__half, true>(a, sign, vec, st) : launch_rotary<__half, false>(a, sign, vec, st);
    else if (dtype == FFNRM_BF16)
        inter ? launch_rotary<__nv_bfloat16, true>(a, sign, vec, st) : launch_rotary<__nv_bfloat16, false>(a, sign, vec, st);
    else
        inter ? launch_rotary<float, true>(a, sign, vec, st) : launch_rotary<float, false>(a, sign, vec, st);
    KV_CUDA(cudaGetLastError());
    return FFNRM_OK;
}

int ffnrm_kv_create(ffnrm_kv **out, int device, const ffnrm_kv_config *cfg, int8_t *k_codes, int8_t *v_codes,
                    float *k_scale, float *v_scale) {
    if (!out || !cfg) return fail(FFNRM_ERR_ARG, "null argument");
    *out = nullptr;
    const ffnrm_kv_config &c = *cfg;
    if (c.n_layers <= 0 || c.kv_heads <= 0 || c.kv_heads > 1024)
        return fail(FFNRM_ERR_ARG, "n_layers=%d must be positive, kv_heads=%d in [1, 1024]", c.n_layers, c.kv_heads);
    if (c.n_pages <= 0 || c.n_pages > (1 << 20)) return fail(FFNRM_ERR_ARG, "n_pages=%d outside [1, 1048576]", c.n_pages);
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256)
        return fail(FFNRM_ERR_ARG, "head_dim=%d must be 64, 128 or 256", c.head_dim);
    if (c.page_tokens != 16 && c.page_tokens != 32 && c.page_tokens != 64 && c.page_tokens != 128)
        return fail(FFNRM_ERR_ARG, "page_tokens=%d must be 16, 32, 64 or 128", c.page_tokens);
    static_assert(kFewSeqs == 4096, "the few-rows kernel keeps a sum for each 32 sequences");
    if (c.max_seqs <= 0 || c.max_seqs > 4096) return fail(FFNRM_ERR_ARG, "max_seqs=%d outside [1, 4096]", c.max_seqs);
    if (!k_codes || !v_codes || !k_scale || !v_scale) return fail(FFNRM_ERR_ARG, "null pool");
    if (!aligned(k_codes, 16) || !aligned(v_codes, 16) || !aligned(k_scale, 4) || !aligned(v_scale, 4))
        return fail(FFNRM_ERR_ARG, "code pools must be 16-byte aligned, scale pools 4-byte");
    ffnrm_kv *kv = new (std::nothrow) ffnrm_kv;
    if (!kv) return fail(FFNRM_ERR_NOMEM, "out of host memory");
    kv->device = device;
    kv->cfg = c;
    while ((1 << kv->page_shift) < c.page_tokens) ++kv->page_shift;
    kv->k_codes = k_codes;
    kv->v_codes = v_codes;
    kv->k_scale = k_scale;
    kv->v_scale = v_scale;
    int count = 0;
    if (cudaGetDeviceCount(&count) != cudaSuccess || device < 0 || device >= count) {
        cudaGetLastError();
        delete kv;
        return fail(FFNRM_ERR_CUDA, "no CUDA device %d", device);
    }
    DeviceGuard guard(device);
    int rc = device_setup(device, kv->setup);
    if (rc) {
        delete kv;
        return rc;
    }
    kv->num_sms = kv->setup->sms;
    // one allocation: page lists, the words that must start as zero (status, arrivals), partials
    const size_t list = size_t(std::max(c.n_pages, c.max_seqs)), lists = 4 * list * sizeof(int32_t);
    int most = 1;
    for (int dtype : {FFNRM_F16, FFNRM_BF16})
        for (int nt : {0, 1}) most = std::max(most, kv->setup->grid[dtype][dim_index(c.head_dim)][nt]);
    const size_t zeros = (size_t(most) + 2) * sizeof(int), partial_at = (lists + zeros + 255) / 256 * 256;
    const size_t bytes = partial_at + kv->setup->floats[dim_index(c.head_dim)] * sizeof(float);
    if (cudaMalloc(&kv->scratch, bytes) != cudaSuccess) {
        cudaGetLastError();
        delete kv;
        return fail(FFNRM_ERR_NOMEM, "cudaMalloc of %zu bytes failed", bytes);
    }
    kv->src = static_cast<int32_t *>(kv->scratch);
    kv->dst = kv->src + list;
    kv->owner = kv->dst + list;
    kv->list = kv->owner + list;
    kv->count = kv->list + list;
    kv->status = kv->count + 1;
    kv->counters = kv->status + 1;
    kv->partial = reinterpret_cast<float *>(static_cast<char *>(kv->scratch) + partial_at);
    cudaError_t e = cudaMemset(kv->count, 0, zeros);
    if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);  // the calls' streams may not be ordered behind it
    if (e != cudaSuccess) {
        cudaFree(kv->scratch);
        delete kv;
        return fail(FFNRM_ERR_CUDA, "creating the cache failed: %s", cudaGetErrorString(e));
    }
    *out = kv;
    return FFNRM_OK;
}

int ffnrm_kv_destroy(ffnrm_kv *kv) {
    if (!kv) return FFNRM_OK;
    DeviceGuard guard(kv->device);
    cudaFree(kv->scratch);  // waits for the device
    cudaGetLastError();
    delete kv;
    return FFNRM_OK;
}

int ffnrm_kv_append(ffnrm_kv *kv, int layer, const ffnrm_kv_batch *batch, int dtype, const ffnrm_rows *k,
                    const ffnrm_rows *v, const ffnrm_rows *q, const ffnrm_rows *q_out, int q_heads, const float *table,
                    int rotary_dim, int max_positions, int flags, void *stream) {
    int rc = check_kv(kv, layer);
    if (rc || (rc = check_batch(kv, batch))) return rc;
    if (dtype < FFNRM_F16 || dtype > FFNRM_F32) return fail(FFNRM_ERR_ARG, "unknown element type %d", dtype);
    const int D = kv->cfg.head_dim;
    if (table && (rc = check_table(table, rotary_dim, max_positions, D, flags, FFNRM_ROTARY_INTERLEAVED))) return rc;
    const bool has_q = q && q->data;
    if (has_q && !table) return fail(FFNRM_ERR_ARG, "q is only rotated: it needs a rotary table");
    if (has_q && q_heads <= 0) return fail(FFNRM_ERR_ARG, "q_heads=%d must be positive", q_heads);
    if (batch->rows == 0 || (batch->seqs == 0 && !has_q)) return FFNRM_OK;
    if (batch->seqs == 0) return fail(FFNRM_ERR_ARG, "rows=%d of no sequence", batch->rows);
    if ((rc = check_rows("k", k, dtype)) || (rc = check_rows("v", v, dtype))) return rc;
    if (has_q) {
        if ((rc = check_rows("q_out", q_out, dtype)) || (rc = check_rows("q", q, dtype))) return rc;
        const size_t size = type_size(dtype);
        if ((rc = check_written("q_out", *q_out, "q", *q, RowPair{batch->rows, q_heads, q_heads, D, size}))) return rc;
        const RowPair kv_pair{batch->rows, kv->cfg.kv_heads, q_heads, D, size};
        if (rows_meet(*k, *q_out, kv_pair) || rows_meet(*v, *q_out, kv_pair)) return fail(FFNRM_ERR_ARG, "q_out must lie apart from k and v");
    }
    const bool inter = flags & FFNRM_ROTARY_INTERLEAVED;
    const int N = 16 / int(type_size(dtype));
    const int T = batch->rows, H = kv->cfg.kv_heads;
    const bool vec = wide(*k, dtype, T, H) && wide(*v, dtype, T, H) &&
                     (!has_q || (wide(*q, dtype, T, q_heads) && wide(*q_out, dtype, T, q_heads))) &&
                     (!table || rotary_fits(inter, 8, D, rotary_dim, table));
    AppendArgs a{};
    a.pool = layer_pool(kv, layer);
    a.batch = batch_view(batch);
    a.k = k->data, a.k_token = k->token_stride, a.k_head = k->head_stride;
    a.v = v->data, a.v_token = v->token_stride, a.v_head = v->head_stride;
    a.table = table, a.rot = table ? rotary_dim : 0, a.max_positions = max_positions;
    a.slots = append_slots(batch->seqs, batch->rows, kv->page_shift, batch->starts != nullptr);
    a.status = kv->status;
    int64_t grid = int64_t(a.slots) * kv->cfg.kv_heads * 2;
    if (has_q) {
        a.q = q->data, a.q_token = q->token_stride, a.q_head = q->head_stride;
        a.q_out = q_out->data, a.o_token = q_out->token_stride, a.o_head = q_out->head_stride;
        a.q_heads = q_heads;
        const int units = vec ? (inter ? D : D - rotary_dim / 2) / N : rotary_units<false, 1>(D, rotary_dim);
        grid += (int64_t(batch->rows) * units * ((q_heads + kQueryHeads - 1) / kQueryHeads) + 255) / 256;
    }
    if (grid > 0x7fffffff) return fail(FFNRM_ERR_ARG, "rows=%d are too many for one call", batch->rows);
    DeviceGuard guard(kv->device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == FFNRM_F16)
        launch_append<__half>(a, vec, inter, unsigned(grid), st);
    else if (dtype == FFNRM_BF16)
        launch_append<__nv_bfloat16>(a, vec, inter, unsigned(grid), st);
    else
        launch_append<float>(a, vec, inter, unsigned(grid), st);
    KV_CUDA(cudaGetLastError());
    return FFNRM_OK;
}

int ffnrm_kv_read(ffnrm_kv *kv, int layer, const ffnrm_kv_batch *batch, int dtype, void *k, void *v, void *stream) {
    int rc = check_kv(kv, layer);
    if (rc || (rc = check_batch(kv, batch))) return rc;
    if (dtype < FFNRM_F16 || dtype > FFNRM_F32) return fail(FFNRM_ERR_ARG, "unknown element type %d", dtype);
    if (batch->rows == 0) return FFNRM_OK;
    if (batch->seqs == 0) return fail(FFNRM_ERR_ARG, "rows=%d of no sequence", batch->rows);
    if (!k || !v || !aligned(k, 32) || !aligned(v, 32)) return fail(FFNRM_ERR_ARG, "k and v must be 32-byte aligned");
    const ReadArgs a{layer_pool(kv, layer), batch_view(batch), k, v, kv->status};
    DeviceGuard guard(kv->device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == FFNRM_F16)
        read_kernel<__half><<<unsigned((batch->rows + 7) / 8), 256, 0, st>>>(a);
    else if (dtype == FFNRM_BF16)
        read_kernel<__nv_bfloat16><<<unsigned((batch->rows + 7) / 8), 256, 0, st>>>(a);
    else
        read_kernel<float><<<unsigned((batch->rows + 7) / 8), 256, 0, st>>>(a);
    KV_CUDA(cudaGetLastError());
    return FFNRM_OK;
}

int ffnrm_kv_attend(ffnrm_kv *kv, int layer, const ffnrm_kv_batch *batch, int dtype, const ffnrm_rows *q,
                    const ffnrm_rows *out, float *lse, int q_heads, float scale, int causal, int window, void *stream) {
    int rc = check_kv(kv, layer);
    if (rc || (rc = check_batch(kv, batch))) return rc;
    if (dtype != FFNRM_F16 && dtype != FFNRM_BF16) return fail(FFNRM_ERR_ARG, "q and out are f16 or bf16, got type %d", dtype);
    if (q_heads <= 0 || q_heads % kv->cfg.kv_heads)
        return fail(FFNRM_ERR_ARG, "q_heads=%d must be a multiple of kv_heads=%d", q_heads, kv->cfg.kv_heads);
    if (window < 0) return fail(FFNRM_ERR_ARG, "window=%d must not be negative", window);
    if (!(scale == scale) || scale <= 0.f || scale > 3.4e38f) return fail(FFNRM_ERR_ARG, "scale must be positive and finite");
    if (batch->rows == 0) return FFNRM_OK;
    if (batch->seqs == 0) return fail(FFNRM_ERR_ARG, "rows=%d of no sequence", batch->rows);
    if ((rc = check_rows("q", q, dtype)) || (rc = check_rows("out", out, dtype))) return rc;
    if (!wide(*q, dtype, batch->rows, q_heads) || !wide(*out, dtype, batch->rows, q_heads))
        return fail(FFNRM_ERR_ARG, "q and out rows must be 16-byte aligned");
    if (!aligned(lse, 4)) return fail(FFNRM_ERR_ARG, "lse must be 4-byte aligned");
    const RowPair pair{batch->rows, q_heads, q_heads, kv->cfg.head_dim, type_size(dtype)};
    if ((rc = check_written("out", *out, "q", *q, pair))) return rc;
    if (lse)
        for (const ffnrm_rows *r : {q, out}) {
            uintptr_t lo, hi;
            extent(*r, batch->rows, q_heads, pair, lo, hi);
            if (share_bytes(lse, size_t(batch->rows) * q_heads * 4, reinterpret_cast<const void *>(lo), hi - lo))
                return fail(FFNRM_ERR_ARG, "lse must lie apart from q and out");
        }
    window = std::min(window, 1 << 30);  // no sequence is longer; keeps position - window in 32 bits
    const AttendArgs a{layer_pool(kv, layer), batch_view(batch), q->data, out->data, lse, q->token_stride, q->head_stride,
                       out->token_stride, out->head_stride, q_heads / kv->cfg.kv_heads, scale, causal, window, kv->status};
    if (int64_t(batch->rows) * a.group > 0x7fffffff / 2)
        return fail(FFNRM_ERR_ARG, "rows=%d are too many for one call", batch->rows);
    DeviceGuard guard(kv->device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // Without starts every sequence has one token; with them the device knows which kernel a sequence takes.
    const int most = few_rows(kv, batch, a.group);
    const bool can_be_many = batch->starts && int64_t(batch->rows) * a.group > most;
    const bool only_many = can_be_many && batch->seqs == 1;
    if (!only_many && (rc = launch_few(kv, a, dtype, can_be_many ? most : 0x7fffffff, st))) return rc;
    return can_be_many ? launch_many(kv, a, dtype, only_many ? 0 : most, only_many, st) : FFNRM_OK;
}

int ffnrm_kv_fork(ffnrm_kv *kv, const int32_t *tables, const int32_t *lengths, int seqs, int table_width,
                  const int32_t *parents, const int32_t *extra, int children, int32_t *out_tables, int out_width,
                  int32_t *out_lengths, int32_t *info, void *stream) {
    if (!kv) return fail(FFNRM_ERR_ARG, "null cache");
    if (seqs < 0 || seqs > kv->cfg.max_seqs || children < 0 || children > kv->cfg.max_seqs)
        return fail(FFNRM_ERR_ARG, "seqs=%d and children=%d must lie in [0, max_seqs=%d]", seqs, children, kv->cfg.max_seqs);
    if (table_width < 0 || out_width < 0 || (int64_t(std::max(table_width, out_width)) << kv->page_shift) > (int64_t(1) << 30))
        return fail(FFNRM_ERR_ARG, "table widths %d and %d must address at most 2^30 tokens", table_width, out_width);
    if (!info || (children && (!parents || !extra || !out_lengths || (out_width && !out_tables))) ||
        (seqs && (!lengths || (table_width && !tables))))
        return fail(FFNRM_ERR_ARG, "null device pointer");
    const size_t table_bytes = size_t(seqs) * table_width * 4, out_bytes = size_t(children) * out_width * 4, length_bytes = size_t(children) * 4;
    if (share_bytes(out_tables, out_bytes, tables, table_bytes)) return fail(FFNRM_ERR_ARG, "out_tables must not lie on the input tables");
    if (share_bytes(out_tables, out_bytes, out_lengths, length_bytes) || share_bytes(info, 16, out_tables, out_bytes) ||
        share_bytes(info, 16, out_lengths, length_bytes))
        return fail(FFNRM_ERR_ARG, "out_tables, out_lengths and info must not lie on one another");
    DeviceGuard guard(kv->device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const PageArgs a{tables, lengths, parents, extra, out_tables, out_lengths, info, kv->src, kv->dst, kv->count, kv->owner,
                     kv->list, seqs, table_width, children, out_width, kv->cfg.n_pages, kv->page_shift, kv->status};
    fork_kernel<<<1, kPageThreads, size_t(kv->cfg.n_pages + 31) / 32 * 4 + size_t(children) * 20, st>>>(a);
    KV_CUDA(cudaGetLastError());
    if (children == 0) return FFNRM_OK;
    return launch_moves(kv, kv->src, kv->dst, kv->count, std::min(children, kv->cfg.n_pages), st);
}

int ffnrm_kv_compact(ffnrm_kv *kv, const int32_t *tables, const int32_t *lengths, int seqs, int table_width,
                     int32_t *out_tables, int32_t *info, void *stream) {
    if (!kv) return fail(FFNRM_ERR_ARG, "null cache");
    if (seqs < 0 || seqs > kv->cfg.max_seqs) return fail(FFNRM_ERR_ARG, "seqs=%d outside [0, max_seqs=%d]", seqs, kv->cfg.max_seqs);
    if (table_width < 0 || (int64_t(table_width) << kv->page_shift) > (int64_t(1) << 30))
        return fail(FFNRM_ERR_ARG, "table_width=%d must address at most 2^30 tokens", table_width);
    if (!info || (seqs && (!lengths || (table_width && (!tables || !out_tables)))))
        return fail(FFNRM_ERR_ARG, "null device pointer");
    const size_t table_bytes = size_t(seqs) * table_width * 4;
    if (out_tables != tables && share_bytes(out_tables, table_bytes, tables, table_bytes))
        return fail(FFNRM_ERR_ARG, "out_tables must be the input tables or lie apart from them");
    if (share_bytes(info, 16, out_tables, table_bytes)) return fail(FFNRM_ERR_ARG, "out_tables and info must not lie on one another");
    DeviceGuard guard(kv->device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const PageArgs a{tables, lengths, nullptr, nullptr, out_tables, nullptr, info, kv->src, kv->dst, kv->count, kv->owner,
                     kv->list, seqs, table_width, 0, table_width, kv->cfg.n_pages, kv->page_shift, kv->status};
    compact_kernel<<<1, kPageThreads, size_t(kv->cfg.n_pages + 31) / 32 * 4 + size_t(seqs) * 4, st>>>(a);
    KV_CUDA(cudaGetLastError());
    return launch_moves(kv, kv->src, kv->dst, kv->count, kv->cfg.n_pages, st);
}

int ffnrm_kv_copy_pages(ffnrm_kv *kv, const int32_t *src, const int32_t *dst, int n, void *stream) {
    if (!kv) return fail(FFNRM_ERR_ARG, "null cache");
    if (n < 0 || n > kv->cfg.n_pages) return fail(FFNRM_ERR_ARG, "n=%d outside [0, n_pages=%d]", n, kv->cfg.n_pages);
    if (n == 0) return FFNRM_OK;
    if (!src || !dst || !aligned(src, 4) || !aligned(dst, 4)) return fail(FFNRM_ERR_ARG, "null or misaligned page lists");
    DeviceGuard guard(kv->device);
    return launch_moves(kv, src, dst, nullptr, n, static_cast<cudaStream_t>(stream));
}

int ffnrm_kv_check(ffnrm_kv *kv, void *stream) {
    if (!kv) return fail(FFNRM_ERR_ARG, "null cache");
    DeviceGuard guard(kv->device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int bits = 0;
    KV_CUDA(cudaMemcpyAsync(&bits, kv->status, sizeof(int), cudaMemcpyDeviceToHost, st));
    KV_CUDA(cudaStreamSynchronize(st));
    if (!bits) return FFNRM_OK;
    KV_CUDA(cudaMemsetAsync(kv->status, 0, sizeof(int), st));
    KV_CUDA(cudaStreamSynchronize(st));
    if (bits & kStatusWait) return fail(FFNRM_ERR_TIMEOUT, "a kernel gave up waiting on a pipeline barrier");
    if (bits & (kStatusPage | kStatusLength | kStatusRotary))
        return fail(FFNRM_ERR_STATE, "a step's data could not be used:%s%s%s",
                    bits & kStatusPage ? " a page id outside the pool;" : "",
                    bits & kStatusLength ? " lengths, rows or room that do not fit the tables or the rows;" : "",
                    bits & kStatusRotary ? " a position past the rotary table;" : "");
    return fail(FFNRM_ERR_NOMEM, "not enough free pages: nothing was forked");
}

}  // extern "C"
