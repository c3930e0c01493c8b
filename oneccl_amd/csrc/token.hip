// Entry points of the token operators (sort, dispatch, combine and its gradient) in libmi_ccl_comp.so.
#include <hip/hip_runtime.h>

#include "../../include/mi_ccl_comp.h"
#include "fusion_plan.hpp"
#include "token_kernels.hpp"

using namespace mi;

namespace {

constexpr uint64_t kMaxRows = 0x7fffffffull;       // positions are int32

bool float_type(int dtype) {
    return dtype == MI_CCL_FLOAT32 || dtype == MI_CCL_FLOAT16 || dtype == MI_CCL_BFLOAT16;
}

// n_tokens x top_k entries and an upper bound of the sorted buffer's rows; false where they do not fit
bool token_sizes(size_t n_tokens, int top_k, int n_experts, size_t align, size_t capacity, uint64_t* entries, uint64_t* rows) {
    if (top_k < 1 || n_experts < 1 || n_experts > kSortMaxExperts || align < 1 || align > kMaxRows || capacity > kMaxRows ||
        n_tokens > kMaxRows / (uint64_t)top_k)
        return false;
    *entries = (uint64_t)n_tokens * (uint64_t)top_k;
    uint64_t kept = *entries;
    if (capacity && capacity * (uint64_t)n_experts < kept) kept = capacity * (uint64_t)n_experts;
    // an expert with rows is padded by at most align - 1
    const uint64_t padded = kept < (uint64_t)n_experts ? kept : (uint64_t)n_experts;
    *rows = kept + padded * (align - 1);
    return *rows <= kMaxRows;
}

bool row_pointer_ok(const void* p, int dtype) {
    return p && (uintptr_t)p % fusion_dtype_size(dtype) == 0;
}

// positions, counts, offsets and fp32 weights, some of which may be NULL
bool words_aligned(const void* a, const void* b = nullptr, const void* c = nullptr, const void* d = nullptr, const void* e = nullptr) {
    return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d | (uintptr_t)e) & 3u) == 0;
}

// How rows of `hidden` elements are shared out: U vectors per lane and one, two or four waves per column tile, the most that leave no
// more lanes without a vector than one wave per tile does; a row's tiles are side by side in the grid.  combine, 16,384 tokens x
// 8 rows of 10 KiB: 250 us in five tiles of 2 KiB, 320 in one of 8 KiB and a quarter of another; rows of 14 KiB 349 and 383.  Where there
// are too few tokens to fill the chip, the most waves that a row fills (dispatch of 7 x 8 rows of 14 KiB 3.9 us, 4.3 in narrow tiles).
RowShape row_shape(size_t hidden, int dtype, size_t n_tokens, int top_k, int u) {
    RowShape s;
    const uint32_t vec = 16 / (uint32_t)fusion_dtype_size(dtype);
    s.nvec = (uint32_t)(hidden / vec);
    s.tail = (uint32_t)(hidden % vec);
    s.log_waves = 0;
    const uint32_t wave = 64u * u, tiles = (s.nvec + wave - 1) / wave;
    while (s.log_waves < 2 && (n_tokens < 256 ? (1u << s.log_waves) < tiles : tiles && tiles % (2u << s.log_waves) == 0)) s.log_waves++;
    const uint32_t width = (64u << s.log_waves) * u;
    s.cols = s.nvec ? (s.nvec + width - 1) / width : 1;
    s.top_k = (uint32_t)top_k;
    s.tokens = n_tokens;
    return s;
}

// Blocks along y, which HIP limits to 65535, and along x: a block takes more tokens, or column tiles, beyond.  The blocks that
// clear the padding come on top (1024 * kPadParts at most).
uint32_t token_blocks(const RowShape& s) {
    constexpr uint64_t kLimit = 65535 - (uint64_t)kSortMaxExperts * kPadParts;
    const uint64_t per_block = (kBlock / 64) >> s.log_waves;
    const uint64_t b = (s.tokens + per_block - 1) / per_block;
    return (uint32_t)(b < kLimit ? b : kLimit);
}
uint32_t column_blocks(const RowShape& s) {
    return s.cols < (1u << 20) ? s.cols : 1u << 20;
}

int launched(const char* name) {
    g_last_kernel = name;
    return fusion_status_of(hipGetLastError());
}

template <class I>
int sort_launch(const I* ids, uint32_t n, uint32_t experts, uint32_t align, uint32_t capacity, int32_t* positions, int32_t* counts,
                int32_t* offsets, uint32_t* table, hipStream_t stream) {
    const SortShape s = sort_shape(n, experts);
    if (s.runs > 1) {
        hipLaunchKernelGGL((token_count_kernel<I>), dim3(s.runs), dim3(kSortBlock), 0, stream, ids, n, experts, s.run, table);
        const int rc = launched("token_count_kernel");
        if (rc != MI_CCL_SUCCESS) return rc;
    }
    if (experts <= 256)
        hipLaunchKernelGGL((token_place_kernel<I, 256>), dim3(s.runs), dim3(kSortBlock), 0, stream, ids, n, experts, s.run, s.runs,
                           (const uint32_t*)table, align, capacity, positions, counts, offsets);
    else
        hipLaunchKernelGGL((token_place_kernel<I, kSortMaxExperts>), dim3(s.runs), dim3(kSortBlock), 0, stream, ids, n, experts, s.run, s.runs,
                           (const uint32_t*)table, align, capacity, positions, counts, offsets);
    return launched("token_place_kernel");
}

// Vectors of a row that a lane takes at once.  16,384 tokens x 8 rows of 8 KiB: dispatch 261 us with one, 264 with two, 278 with
// four (a wave's stores go to eight places; more of them at once only mix more); combine 207, 203 and 205.  Rows that one vector per lane
// of a wave covers are combined with one (rows of 1 KiB: 31 us, 35 with two).
constexpr int kDispatchU = 1;
int combine_u(size_t hidden, int dtype) {
    return hidden * fusion_dtype_size(dtype) <= 64 * 16 ? 1 : 2;
}

template <class E>
void dispatch_launch(const RowShape& s, uint32_t experts, hipStream_t stream, const void* x, size_t ld_x, const int32_t* positions,
                     const int32_t* counts, const int32_t* offsets, void* out, size_t ld_out, size_t rows) {
    hipLaunchKernelGGL((token_dispatch_kernel<E, kDispatchU>), dim3(column_blocks(s), pad_blocks(experts) + token_blocks(s)), dim3(kBlock), 0, stream,
                       (const unsigned char*)x, (uint64_t)ld_x, s, experts, positions, counts, offsets, (unsigned char*)out, (uint64_t)ld_out, (uint64_t)rows);
}

template <class V, int U, int K>
void combine_launch(const RowShape& s, hipStream_t stream, const void* y, size_t ld_y, size_t rows, const int32_t* positions,
                    const float* weights, void* out, size_t ld_out) {
    hipLaunchKernelGGL((token_combine_kernel<V, U, K>), dim3(column_blocks(s), token_blocks(s)), dim3(kBlock), 0, stream, (const unsigned char*)y,
                       (uint64_t)ld_y, (uint64_t)rows, s, positions, weights, (unsigned char*)out, (uint64_t)ld_out);
}
template <class V, int U>
void combine_by_k(const RowShape& s, hipStream_t stream, const void* y, size_t ld_y, size_t rows, const int32_t* positions,
                  const float* weights, void* out, size_t ld_out) {
    if (s.top_k == 1) combine_launch<V, U, 1>(s, stream, y, ld_y, rows, positions, weights, out, ld_out);
    else if (s.top_k == 2) combine_launch<V, U, 2>(s, stream, y, ld_y, rows, positions, weights, out, ld_out);
    else if (s.top_k <= 4) combine_launch<V, U, 4>(s, stream, y, ld_y, rows, positions, weights, out, ld_out);
    else combine_launch<V, U, 8>(s, stream, y, ld_y, rows, positions, weights, out, ld_out);
}

template <class V>
void combine_by_u(const RowShape& s, int u, hipStream_t stream, const void* y, size_t ld_y, size_t rows, const int32_t* positions,
                  const float* weights, void* out, size_t ld_out) {
    if (u == 1) combine_by_k<V, 1>(s, stream, y, ld_y, rows, positions, weights, out, ld_out);
    else combine_by_k<V, 2>(s, stream, y, ld_y, rows, positions, weights, out, ld_out);
}

struct BackwardArgs {
    RowShape s;
    uint32_t block, grid, experts;
    hipStream_t stream;
    const void *grad, *y;
    size_t ld_grad, ld_y, ld_grad_y, rows;
    const int32_t *positions, *counts, *offsets;
    const float* weights;
    void* grad_y;
    float* grad_weights;
};
template <class V, int K, bool DOT>
void backward_launch(const BackwardArgs& a) {
    hipLaunchKernelGGL((token_combine_backward_kernel<V, K, DOT>), dim3(a.grid), dim3(a.block), 0, a.stream, (const unsigned char*)a.grad,
                       (uint64_t)a.ld_grad, (const unsigned char*)a.y, (uint64_t)a.ld_y, (uint64_t)a.rows, a.s, a.experts, a.positions,
                       a.weights, a.counts, a.offsets, (unsigned char*)a.grad_y, (uint64_t)a.ld_grad_y, a.grad_weights);
}
template <class V, bool DOT>
void backward_by_k(const BackwardArgs& a) {
    if (a.s.top_k == 1) backward_launch<V, 1, DOT>(a);
    else if (a.s.top_k == 2) backward_launch<V, 2, DOT>(a);
    else if (a.s.top_k <= 4) backward_launch<V, 4, DOT>(a);
    else backward_launch<V, 8, DOT>(a);
}
template <class V>
void backward_by_dot(const BackwardArgs& a) {
    if (a.grad_weights) backward_by_k<V, true>(a);
    else backward_by_k<V, false>(a);
}

// ---- rows in the order of the buffer

// Where it pays: from 64 MiB of rows, as far as HIP takes the blocks in one launch.  Against token by token, with buffers that
// the 256 MB cache cannot hold: dispatch of 16,384 tokens x 8 rows of 8 KiB 217 against 247 us, both gradients of 8,192 x 8 291
// against 318; dispatch and combine's gradient of 8,192 x 4 rows of 14 KiB 91 and 172 against 127 and 202, of 65,536 x 1 of 8 KiB
// 184 and 267 against 186 and 301.  At 33 MiB (2,048 x 2 of 8 KiB) the launch in front costs what it gains: 13 and 20 us
// against 11 and 19.  "variant" 8 takes it at any size.
constexpr uint64_t kOrderBytes = 64u << 20;
bool wants_order(int dtype, size_t n_tokens, int top_k, size_t hidden) {
    const uint64_t entries = (uint64_t)n_tokens * (uint64_t)top_k;
    if (entries == 0 || hidden == 0 || entries >= (1u << 22))
        return false;
    return entries * hidden * fusion_dtype_size(dtype) >= kOrderBytes || mi_ccl_get_param("variant") == 8;
}
// Lanes of an entry, whole waves, 64 to 512.  Dispatch has one load and one store per vector: as many lanes as the row has
// vectors (16,384 tokens x 8 rows of 320 vectors: 112 us with 320 lanes, 133 with 512, 124 with 192 twice round; of 160 vectors 60 with
// 192, 70 with 256).  The gradient, which has more to do per vector, takes a power of two and lets a third of the lanes go round twice:
// 160 vectors 127 us with 128 lanes, 130 with 192; 320 vectors 234 with 256, 252 with 320; 26,296 x 5 rows of 139 vectors 158 with
// 128, 206 with 256.  Up to 128 lanes a block of 256 takes several entries (26,296 x 8 rows of 64 vectors: dispatch 40 us, 51 in
// blocks of 64).
uint32_t order_lanes(uint32_t nvec, bool one_each) {
    if (one_each) return nvec <= 64 ? 64u : nvec < 512 ? (nvec + 63) / 64 * 64 : 512u;
    uint32_t lanes = 64;
    while (lanes < 512 && lanes + lanes / 2 < nvec) lanes <<= 1;
    return lanes;
}
// Entries per run: what keeps the run's tokens within 2 MiB, half of an XCD's L2, and leaves no XCD without a run in a tenth of the
// turns (an XCD takes every eighth run).  Dispatch, two buffer sets in turn: 16,384 tokens x 8 of 8 KiB 184 us with 2,048 entries, 190 with
// 1,024, 193 with 512, 201 with 256; 8,192 x 4 of 14 KiB 116, 93, 91, 90; 5,000 x 8 of 8 KiB, 20 runs of 2,048 or 40 of 1,024, 67 and 60;
// 2,304 x 8, 9 runs of 2,048 or 36 of 512, 42 and 30.
uint32_t order_log_run(uint64_t entries, uint32_t top_k, uint64_t row_bytes) {
    uint32_t log_run = 8;
    while (log_run < 11 && ((2ull << log_run) / top_k) * row_bytes <= (2u << 20)) log_run++;
    for (; log_run > 8; log_run--) {
        const uint64_t runs = (entries + (1u << log_run) - 1) >> log_run, turns = (runs + 7) / 8;
        if (10 * runs >= 9 * 8 * turns) break;
    }
    return log_run;
}
constexpr uint32_t kOrderMulti = 128;        // lanes of an entry up to which a block takes several (64 or 128: powers of two)
uint32_t order_blocks(uint64_t entries, uint32_t log_run, uint32_t lanes) {         // eight runs at a time
    const uint64_t runs = (entries + (1u << log_run) - 1) >> log_run;
    return (uint32_t)((((runs + 7) / 8 * 8) << log_run) / (lanes <= kOrderMulti ? kOrderedMultiBlock / lanes : 1));
}
int order_launch(const int32_t* positions, uint64_t entries, uint32_t log_run, size_t rows, OrderedEntry* order, hipStream_t stream) {
    uint32_t shift = 0;
    while (((uint64_t)(rows - 1) >> shift) >= kOrderBuckets) shift++;
    hipLaunchKernelGGL(token_order_kernel, dim3((unsigned)((entries + (1u << log_run) - 1) >> log_run)), dim3(kOrderBlock), 0, stream, positions,
                       entries, 1u << log_run, (uint64_t)rows, shift, order);
    return launched("token_order_kernel");
}

struct OrderedArgs {
    dim3 grid, block;
    hipStream_t stream;
    uint32_t experts, log_lanes, log_run;       // log_lanes: of several entries per block
    uint64_t entries;
    const OrderedEntry* order;
    bool multi;
    OrderedArgs(uint32_t lanes, uint32_t experts_, uint32_t log_run_, uint64_t entries_, const OrderedEntry* order_, hipStream_t stream_)
        : grid(pad_blocks(experts_) + order_blocks(entries_, log_run_, lanes)), block(lanes <= kOrderMulti ? kOrderedMultiBlock : lanes),
          stream(stream_), experts(experts_), log_lanes(lanes == 64 ? 6 : 7), log_run(log_run_), entries(entries_), order(order_),
          multi(lanes <= kOrderMulti) {}
};
template <class E, bool MULTI>
void dispatch_ordered_launch(const OrderedArgs& o, const RowShape& s, const void* x, size_t ld_x, const int32_t* counts, const int32_t* offsets,
                             void* out, size_t ld_out, size_t rows) {
    hipLaunchKernelGGL((token_dispatch_ordered_kernel<E, MULTI>), o.grid, o.block, 0, o.stream, (const unsigned char*)x, (uint64_t)ld_x, s.nvec, s.tail,
                       s.top_k, o.entries, o.experts, o.order, o.log_lanes, o.log_run, counts, offsets, (unsigned char*)out, (uint64_t)ld_out,
                       (uint64_t)rows);
}
template <class E>
void dispatch_ordered(const OrderedArgs& o, const RowShape& s, const void* x, size_t ld_x, const int32_t* counts, const int32_t* offsets, void* out,
                      size_t ld_out, size_t rows) {
    if (o.multi) dispatch_ordered_launch<E, true>(o, s, x, ld_x, counts, offsets, out, ld_out, rows);
    else dispatch_ordered_launch<E, false>(o, s, x, ld_x, counts, offsets, out, ld_out, rows);
}

template <class V, bool DOT, bool MULTI>
void backward_ordered_launch(const OrderedArgs& o, const BackwardArgs& a) {
    hipLaunchKernelGGL((token_backward_ordered_kernel<V, DOT, MULTI>), o.grid, o.block, 0, o.stream, (const unsigned char*)a.grad, (uint64_t)a.ld_grad,
                       (const unsigned char*)a.y, (uint64_t)a.ld_y, a.s.nvec, a.s.tail, a.s.top_k, o.entries, o.experts, o.order, o.log_lanes, o.log_run,
                       a.weights, a.counts, a.offsets, (unsigned char*)a.grad_y, (uint64_t)a.ld_grad_y, (uint64_t)a.rows, a.grad_weights);
}
template <class V, bool DOT>
void backward_ordered(const BackwardArgs& a, const OrderedEntry* order, uint32_t log_run) {
    const uint64_t entries = a.s.tokens * a.s.top_k;
    const OrderedArgs o(order_lanes(a.s.nvec, false), a.experts, log_run, entries, order, a.stream);
    if (o.multi) backward_ordered_launch<V, DOT, true>(o, a);
    else backward_ordered_launch<V, DOT, false>(o, a);
}
template <class V>
void backward_ordered_by_dot(const BackwardArgs& a, const OrderedEntry* order, uint32_t log_run) {
    if (a.grad_weights) backward_ordered<V, true>(a, order, log_run);
    else backward_ordered<V, false>(a, order, log_run);
}

}  // namespace

extern "C" {

int mi_ccl_token_order_workspace(int dtype, size_t n_tokens, int top_k, size_t hidden, size_t* bytes) {
    if (!bytes || !float_type(dtype) || top_k < 1 || n_tokens > kMaxRows / (uint64_t)top_k || hidden > kMaxRows)
        return MI_CCL_INVALID_ARGUMENTS;
    *bytes = wants_order(dtype, n_tokens, top_k, hidden) ? n_tokens * (size_t)top_k * sizeof(OrderedEntry) : 0;
    return MI_CCL_SUCCESS;
}

int mi_ccl_token_rows(size_t n_tokens, int top_k, int n_experts, size_t align, size_t capacity, size_t* rows) {
    uint64_t entries = 0, r = 0;
    if (!rows || !token_sizes(n_tokens, top_k, n_experts, align, capacity, &entries, &r))
        return MI_CCL_INVALID_ARGUMENTS;
    *rows = (size_t)r;
    return MI_CCL_SUCCESS;
}

int mi_ccl_token_sort_workspace(size_t n_tokens, int top_k, int n_experts, size_t* bytes) {
    uint64_t entries = 0, r = 0;
    if (!bytes || !token_sizes(n_tokens, top_k, n_experts, 1, 0, &entries, &r))
        return MI_CCL_INVALID_ARGUMENTS;
    const SortShape s = sort_shape((uint32_t)entries, (uint32_t)n_experts);
    *bytes = s.runs > 1 ? (size_t)s.runs * (size_t)n_experts * sizeof(uint32_t) : 0;
    return MI_CCL_SUCCESS;
}

int mi_ccl_token_sort(int index_dtype, const void* expert_ids, size_t n_tokens, int top_k, int n_experts, size_t align, size_t capacity,
                      int32_t* positions, int32_t* counts, int32_t* offsets, void* workspace, size_t workspace_bytes, void* stream) {
    uint64_t entries = 0, rows = 0;
    size_t need = 0;
    if ((index_dtype != MI_CCL_INT32 && index_dtype != MI_CCL_INT64) || !counts || !offsets ||
        !token_sizes(n_tokens, top_k, n_experts, align, capacity, &entries, &rows))
        return MI_CCL_INVALID_ARGUMENTS;
    if (entries && (!expert_ids || (uintptr_t)expert_ids % fusion_dtype_size(index_dtype) || !positions))
        return MI_CCL_INVALID_ARGUMENTS;
    if (!words_aligned(positions, counts, offsets, workspace))
        return MI_CCL_INVALID_ARGUMENTS;
    mi_ccl_token_sort_workspace(n_tokens, top_k, n_experts, &need);
    if (need && (!workspace || workspace_bytes < need))
        return MI_CCL_INVALID_ARGUMENTS;
    const uint32_t cap = capacity ? (uint32_t)capacity : 0xffffffffu;
    if (index_dtype == MI_CCL_INT32)
        return sort_launch<int32_t>((const int32_t*)expert_ids, (uint32_t)entries, (uint32_t)n_experts, (uint32_t)align, cap, positions, counts,
                                    offsets, (uint32_t*)workspace, (hipStream_t)stream);
    return sort_launch<int64_t>((const int64_t*)expert_ids, (uint32_t)entries, (uint32_t)n_experts, (uint32_t)align, cap, positions, counts,
                                offsets, (uint32_t*)workspace, (hipStream_t)stream);
}

int mi_ccl_token_dispatch(int dtype, const void* x, size_t ld_x, size_t n_tokens, int top_k, size_t hidden, const int32_t* positions,
                          const int32_t* counts, const int32_t* offsets, int n_experts, void* out, size_t ld_out, size_t out_rows,
                          void* workspace, size_t workspace_bytes, void* stream) {
    if (!float_type(dtype) || top_k < 1 || n_experts < 1 || n_experts > kSortMaxExperts)
        return MI_CCL_INVALID_ARGUMENTS;
    if (n_tokens == 0 || hidden == 0 || out_rows == 0)
        return MI_CCL_SUCCESS;
    if (!row_pointer_ok(x, dtype) || !row_pointer_ok(out, dtype) || !positions || !counts || !offsets || ld_x < hidden || ld_out < hidden ||
        hidden > kMaxRows || n_tokens > kMaxRows / (uint64_t)top_k || out_rows > kMaxRows || !words_aligned(positions, counts, offsets))
        return MI_CCL_INVALID_ARGUMENTS;
    if ((uintptr_t)workspace % sizeof(OrderedEntry))
        return MI_CCL_INVALID_ARGUMENTS;
    const RowShape s = row_shape(hidden, dtype, n_tokens, top_k, kDispatchU);
    const uint64_t entries = (uint64_t)n_tokens * (uint64_t)top_k;
    if (workspace && workspace_bytes / sizeof(OrderedEntry) >= entries && wants_order(dtype, n_tokens, top_k, hidden)) {
        OrderedEntry* order = (OrderedEntry*)workspace;
        const uint32_t log_run = order_log_run(entries, s.top_k, hidden * fusion_dtype_size(dtype));
        const int rc = order_launch(positions, entries, log_run, out_rows, order, (hipStream_t)stream);
        if (rc != MI_CCL_SUCCESS)
            return rc;
        const OrderedArgs o(order_lanes(s.nvec, true), (uint32_t)n_experts, log_run, entries, order, (hipStream_t)stream);
        if (fusion_dtype_size(dtype) == 4) dispatch_ordered<uint32_t>(o, s, x, ld_x, counts, offsets, out, ld_out, out_rows);
        else dispatch_ordered<uint16_t>(o, s, x, ld_x, counts, offsets, out, ld_out, out_rows);
        return launched("token_dispatch_ordered_kernel");
    }
    if (fusion_dtype_size(dtype) == 4)
        dispatch_launch<uint32_t>(s, (uint32_t)n_experts, (hipStream_t)stream, x, ld_x, positions, counts, offsets, out, ld_out, out_rows);
    else
        dispatch_launch<uint16_t>(s, (uint32_t)n_experts, (hipStream_t)stream, x, ld_x, positions, counts, offsets, out, ld_out, out_rows);
    return launched("token_dispatch_kernel");
}

int mi_ccl_token_combine(int dtype, const void* y, size_t ld_y, size_t y_rows, const int32_t* positions, const float* weights,
                         size_t n_tokens, int top_k, size_t hidden, void* out, size_t ld_out, void* stream) {
    if (!float_type(dtype) || top_k < 1)
        return MI_CCL_INVALID_ARGUMENTS;
    if (n_tokens == 0 || hidden == 0)
        return MI_CCL_SUCCESS;
    if ((y_rows && !row_pointer_ok(y, dtype)) || !row_pointer_ok(out, dtype) || !positions || ld_y < hidden || ld_out < hidden ||
        hidden > kMaxRows || n_tokens > kMaxRows / (uint64_t)top_k || y_rows > kMaxRows || !words_aligned(positions, weights))
        return MI_CCL_INVALID_ARGUMENTS;
    const int u = combine_u(hidden, dtype);
    const RowShape s = row_shape(hidden, dtype, n_tokens, top_k, u);
    if (dtype == MI_CCL_FLOAT32) combine_by_u<F32Vec>(s, u, (hipStream_t)stream, y, ld_y, y_rows, positions, weights, out, ld_out);
    else if (dtype == MI_CCL_BFLOAT16) combine_by_u<Bf16Vec>(s, u, (hipStream_t)stream, y, ld_y, y_rows, positions, weights, out, ld_out);
    else combine_by_u<Fp16Vec>(s, u, (hipStream_t)stream, y, ld_y, y_rows, positions, weights, out, ld_out);
    return launched("token_combine_kernel");
}

int mi_ccl_token_combine_backward(int dtype, const void* grad_out, size_t ld_grad, const void* y, size_t ld_y, size_t y_rows,
                                  const int32_t* positions, const float* weights, const int32_t* counts, const int32_t* offsets,
                                  int n_experts, size_t n_tokens, int top_k, size_t hidden, void* grad_y, size_t ld_grad_y,
                                  float* grad_weights, void* workspace, size_t workspace_bytes, void* stream) {
    if (!float_type(dtype) || top_k < 1 || n_experts < 1 || n_experts > kSortMaxExperts)
        return MI_CCL_INVALID_ARGUMENTS;
    if (n_tokens == 0)
        return MI_CCL_SUCCESS;
    if (!positions || !counts || !offsets || hidden > kMaxRows || n_tokens > kMaxRows / (uint64_t)top_k || y_rows > kMaxRows ||
        !words_aligned(positions, weights, counts, offsets, grad_weights) || (uintptr_t)workspace % sizeof(OrderedEntry))
        return MI_CCL_INVALID_ARGUMENTS;
    if (hidden && (!row_pointer_ok(grad_out, dtype) || ld_grad < hidden))
        return MI_CCL_INVALID_ARGUMENTS;
    if (hidden && y_rows && (!row_pointer_ok(grad_y, dtype) || ld_grad_y < hidden || (grad_weights && (!row_pointer_ok(y, dtype) || ld_y < hidden))))
        return MI_CCL_INVALID_ARGUMENTS;
    if (!grad_weights && (hidden == 0 || y_rows == 0))
        return MI_CCL_SUCCESS;
    BackwardArgs a;
    a.s = row_shape(hidden, dtype, n_tokens, top_k, 1);
    // A block per token: as many lanes as the row has vectors, at most 512 (8,192 tokens x 8 rows of 8 KiB, both gradients: 318 us;
    // 321 with 256 lanes, 330 with 128), up to 1024 when there are too few tokens to fill the chip.
    const uint32_t most = n_tokens >= 256 ? 512 : 1024;
    a.block = 64;
    while (a.block < a.s.nvec && a.block < most) a.block <<= 1;
    a.experts = (uint32_t)n_experts;
    a.grid = pad_blocks(a.experts) + (uint32_t)(n_tokens < (1u << 20) ? n_tokens : 1u << 20);
    a.stream = (hipStream_t)stream;
    a.grad = grad_out;
    a.ld_grad = ld_grad;
    a.y = y;
    a.ld_y = ld_y;
    a.rows = y_rows;
    a.positions = positions;
    a.weights = weights;
    a.counts = counts;
    a.offsets = offsets;
    a.grad_y = grad_y;
    a.ld_grad_y = ld_grad_y;
    a.grad_weights = grad_weights;
    const uint64_t entries = (uint64_t)n_tokens * (uint64_t)top_k;
    if (y_rows && workspace && workspace_bytes / sizeof(OrderedEntry) >= entries && wants_order(dtype, n_tokens, top_k, hidden)) {
        const uint32_t log_run = order_log_run(entries, a.s.top_k, hidden * fusion_dtype_size(dtype));
        const int rc = order_launch(positions, entries, log_run, y_rows, (OrderedEntry*)workspace, (hipStream_t)stream);
        if (rc != MI_CCL_SUCCESS)
            return rc;
        if (dtype == MI_CCL_FLOAT32) backward_ordered_by_dot<F32Vec>(a, (const OrderedEntry*)workspace, log_run);
        else if (dtype == MI_CCL_BFLOAT16) backward_ordered_by_dot<Bf16Vec>(a, (const OrderedEntry*)workspace, log_run);
        else backward_ordered_by_dot<Fp16Vec>(a, (const OrderedEntry*)workspace, log_run);
        return launched("token_backward_ordered_kernel");
    }
    if (dtype == MI_CCL_FLOAT32) backward_by_dot<F32Vec>(a);
    else if (dtype == MI_CCL_BFLOAT16) backward_by_dot<Bf16Vec>(a);
    else backward_by_dot<Fp16Vec>(a);
    return launched("token_combine_backward_kernel");
}

} /* extern "C" */
