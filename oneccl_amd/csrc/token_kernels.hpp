// Tokens sorted by the expert they were routed to, copied into one buffer expert after expert (the send buffer of an
// expert-parallel all-to-all, or the operand of the experts' products), and brought back as a weighted sum.
//
// T tokens have k entries each, entry i = t k + j with expert id e(i); ids outside [0, E) are no entry (a masked token).
//   rank(i)    = number of entries i' < i with e(i') = e(i); entries of rank >= capacity are dropped
//   count(e)   = min(entries of e, capacity);  offset(e + 1) = offset(e) + count(e) rounded up to `align`
//   pos(i)     = offset(e(i)) + rank(i), -1 where there is no entry or it is dropped
//   dispatch   : out[pos(t, j)] = x[t];  rows of padding (between count and the next offset) = 0
//   combine    : out[t] = sum_j w(t, j) y[pos(t, j)]
//   its gradient: dy[pos(t, j)] = w(t, j) g[t], dw(t, j) = <g[t], y[pos(t, j)]>
#pragma once

#include "float_vec.hpp"

namespace mi {

// ---- sort ---------------------------------------------------------------------------------------------------------------
// A stable counting sort.  A block of 16 waves takes a contiguous run of entries, a wave a sixteenth of it.  Up to
// kSortSingle entries one block does everything in one launch; beyond, a first launch counts the experts of every run
// (runs x E numbers in the workspace) and in a second every block adds up the runs before its own, which costs each block
// a read of that table and saves the launch of a scan between the two.  What bounds it is latency: the passes of a block over its
// run, and the table, which grows with the number of runs; the two meet at about 2 sqrt(n / E) runs.  Measured as nodes of a
// replayed graph: 2,048 entries 4.9 us, 4,096 6.9, 8,192 7.3 (in one block 11), 131,072 over 128 experts 9.8 (64 runs; 10.9 with 128,
// 11.2 with 32), 524,288 over 256 19.2 (128 runs; 20.2 with 64, 25.3 with 256), 2,097,152 over 128 25 (256 runs; 50 with 64).
constexpr int kSortBlock = 1024;
constexpr int kSortWaves = kSortBlock / 64;
constexpr int kSortMaxExperts = 1024;
constexpr uint32_t kSortSingle = 4096;      // entries one block sorts alone
constexpr uint32_t kSortRun = 2048;         // fewest entries of a block's run

// runs and entries per run of a sort of n entries (a run is a whole number of entries per lane)
struct SortShape {
    uint32_t runs, run;
};
inline SortShape sort_shape(uint32_t n, uint32_t experts) {
    if (n <= kSortSingle) return SortShape{ 1, ((n + kSortBlock - 1) / kSortBlock) * kSortBlock };
    uint32_t runs = 16;
    while (runs < 512 && (uint64_t)runs * runs * experts < 4ull * n) runs++;
    uint32_t run = (uint32_t)(((uint64_t)n + runs - 1) / runs);
    run = (run + kSortBlock - 1) / kSortBlock * kSortBlock;
    if (run < kSortRun) run = kSortRun;
    return SortShape{ (uint32_t)(((uint64_t)n + run - 1) / run), run };
}

// the expert of entry i, or E when it has none
template <class I>
__device__ __forceinline__ uint32_t entry_expert(const I* ids, uint32_t i, uint32_t n, uint32_t experts) {
    if (i >= n) return experts;
    const I e = ids[i];
    return (e >= 0 && e < (I)experts) ? (uint32_t)e : experts;
}

template <class I>
__global__ void __launch_bounds__(kSortBlock)
token_count_kernel(const I* ids, uint32_t n, uint32_t experts, uint32_t run, uint32_t* table) {
    __shared__ uint32_t hist[kSortMaxExperts];
    for (uint32_t e = threadIdx.x; e < experts; e += kSortBlock) hist[e] = 0;
    __syncthreads();
    const uint64_t first = (uint64_t)blockIdx.x * run;
    for (uint32_t o = threadIdx.x; o < run; o += kSortBlock) {
        const uint64_t i = first + o;
        if (i >= n) break;
        const uint32_t e = entry_expert(ids, (uint32_t)i, n, experts);
        if (e < experts) atomicAdd(&hist[e], 1u);       // a count: the order of the additions does not matter
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < experts; e += kSortBlock) table[(size_t)blockIdx.x * experts + e] = hist[e];
}

// LDS: kSortWaves x E wave counts, then E totals and E first rows; MAXE experts at most.
template <class I, int MAXE>
__global__ void __launch_bounds__(kSortBlock)
token_place_kernel(const I* ids, uint32_t n, uint32_t experts, uint32_t run, uint32_t runs, const uint32_t* table, uint32_t align,
                   uint32_t capacity, int32_t* positions, int32_t* counts, int32_t* offsets) {
    __shared__ uint32_t lds[(kSortWaves + 2) * MAXE];
    uint32_t* const wave_count = lds;
    uint32_t* const total = lds + kSortWaves * experts;
    uint32_t* const begin = total + experts;
    __shared__ uint32_t wave_end[kSortWaves];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t per_wave = run / kSortWaves;         // a multiple of 64
    const uint64_t first = (uint64_t)blockIdx.x * run + (uint64_t)wave * per_wave;
    for (uint32_t e = tid; e < (kSortWaves + 2) * experts; e += kSortBlock) lds[e] = 0;
    __syncthreads();

    uint32_t* const mine = wave_count + wave * experts;
    for (uint32_t o = lane; o < per_wave && first + o < n; o += 64) {
        const uint32_t e = entry_expert(ids, (uint32_t)(first + o), n, experts);
        if (e < experts) atomicAdd(&mine[e], 1u);
    }
    __syncthreads();
    // totals of every expert, and how many entries the runs before this one hold (kept in begin[] for now)
    if (runs == 1) {
        for (uint32_t e = tid; e < experts; e += kSortBlock) {
            uint32_t s = 0;
            for (int w = 0; w < kSortWaves; w++) s += wave_count[w * experts + e];
            total[e] = s;
        }
    }
    else {
        // lanes side by side take experts side by side; the rows of the table are shared out over what is left
        uint32_t width = 64;
        while (width < experts && width < (uint32_t)kSortBlock) width <<= 1;
        const uint32_t groups = kSortBlock / width, g = tid / width;
        for (uint32_t e = tid & (width - 1); e < experts; e += width) {
            uint32_t all = 0, before = 0;
            for (uint32_t r = g; r < runs; r += groups) {
                const uint32_t c = table[(size_t)r * experts + e];
                all += c;
                before += r < blockIdx.x ? c : 0u;
            }
            atomicAdd(&total[e], all);
            atomicAdd(&begin[e], before);
        }
    }
    __syncthreads();
    // offsets: the sum of the padded counts before each expert.  Lane e of the block holds expert e (E <= block).
    uint32_t kept = 0, padded = 0;
    if (tid < experts) {
        kept = total[tid] < capacity ? total[tid] : capacity;
        padded = (kept + align - 1) / align * align;
    }
    uint32_t incl = padded;
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint32_t up = __shfl_up(incl, d, 64);
        if (lane >= d) incl += up;
    }
    if (lane == 63) wave_end[wave] = incl;
    __syncthreads();
    uint32_t base = 0;
    for (uint32_t w = 0; w < wave; w++) base += wave_end[w];
    const uint32_t offset = base + incl - padded;
    if (tid < experts) {
        // the rank with which each wave's first entry of this expert starts
        uint32_t rank = begin[tid];
        for (int w = 0; w < kSortWaves; w++) {
            const uint32_t c = wave_count[w * experts + tid];
            wave_count[w * experts + tid] = rank;
            rank += c;
        }
        begin[tid] = offset;
        if (blockIdx.x == 0) {
            counts[tid] = (int32_t)kept;
            offsets[tid] = (int32_t)offset;
            if (tid == experts - 1) offsets[experts] = (int32_t)(offset + padded);
        }
    }
    __syncthreads();
    // 64 entries at a time, in order: the lanes of one expert find each other by the bits of its id
    volatile uint32_t* const next = mine;
    const int bits = 32 - __clz(experts);               // the id E (no entry) takes part
    for (uint32_t o = lane; o < per_wave; o += 64) {
        const uint64_t i = first + o;
        if (first + (o - lane) >= n) break;             // the same answer for the whole wave
        const uint32_t e = i < n ? entry_expert(ids, (uint32_t)i, n, experts) : experts;
        uint64_t same = ~0ull;
        for (int b = 0; b < bits; b++) {
            const bool set = (e >> b) & 1u;
            const uint64_t with = __ballot(set);
            same &= set ? with : ~with;
        }
        const uint32_t before = __popcll(same & ((1ull << lane) - 1));
        uint32_t rank = 0;
        if (e < experts) rank = next[e] + before;
        __builtin_amdgcn_wave_barrier();
        if (e < experts && before == 0) next[e] = rank + __popcll(same);        // the first of them: its rank is the old value
        __builtin_amdgcn_wave_barrier();
        if (i < n) positions[i] = (e < experts && rank < capacity) ? (int32_t)(begin[e] + rank) : -1;
    }
}

// ---- rows ---------------------------------------------------------------------------------------------------------------
// A row of H elements: vectors of 16 bytes, then H % VEC elements.  Rows may start anywhere (H odd, a stride, a slice): the
// vectors are loose.  1 << log_waves waves of a block take one token, and of its vectors the column tiles blockIdx.x,
// blockIdx.x + gridDim.x, ... of (64 << log_waves) U vectors each, so that a row's tiles are neighbours in time; the elements
// behind the last vector belong to the last tile.
struct RowShape {
    uint32_t nvec, tail;        // vectors and elements behind them
    uint32_t cols;              // column tiles, at least 1
    uint32_t log_waves;
    uint32_t top_k;
    uint64_t tokens;
};

// Clears the rows of padding behind one expert's rows, every kPadParts-th of them; pad_blocks(experts) blocks do
// all.  They come first in the grid: behind the tokens' they would be what a launch waits for at its end.  Their number is a
// multiple of the XCDs, so that the block behind them has the first one; with an odd number of experts the last ones are idle.
constexpr uint32_t kPadParts = 4;
__host__ __device__ constexpr uint32_t pad_blocks(uint32_t experts) {
    return (experts * kPadParts + 7) / 8 * 8;
}
template <class E>
__device__ __forceinline__ void clear_padding(uint32_t block, uint32_t experts, const int32_t* counts, const int32_t* offsets, uint64_t rows,
                                              unsigned char* out, uint64_t ld, uint32_t nvec, uint32_t tail) {
    constexpr uint32_t VEC = 16 / sizeof(E);
    const uint32_t expert = block / kPadParts;
    if (expert >= experts) return;
    const int64_t r0 = (int64_t)offsets[expert] + counts[expert];
    int64_t r1 = offsets[expert + 1];
    if (r0 < 0) return;
    if (r1 > (int64_t)rows) r1 = (int64_t)rows;
    for (int64_t r = r0 + block % kPadParts; r < r1; r += kPadParts) {
        unsigned char* o = out + (uint64_t)r * ld * sizeof(E);
        for (uint32_t v = threadIdx.x; v < nvec; v += blockDim.x) st_loose((u32x4_u*)o + v, u32x4{ 0, 0, 0, 0 });
        for (uint32_t i = threadIdx.x; i < tail; i += blockDim.x) st_elem<E>(o, (uint64_t)nvec * VEC + i, (E)0);
    }
}

// Up to K entries of a token: their rows, -1 where there is none (or the position is none of the buffer's rows).
template <int K>
__device__ __forceinline__ void load_positions(const int32_t* pos, uint32_t k, uint64_t rows, int32_t (&p)[K]) {
#pragma unroll
    for (int j = 0; j < K; j++) {
        p[j] = (uint32_t)j < k ? pos[j] : -1;
        if (p[j] >= 0 && (uint64_t)p[j] >= rows) p[j] = -1;
    }
}

// ---- rows in the order of the buffer ----------------------------------------------------------------------------------------
// Dispatch and combine's gradient, token by token, write a token's k rows to k places far apart, and memory takes 8 KiB
// here and 8 KiB there at 5.2 TB/s where a compact window runs at 6.7.  Large calls therefore take runs of 256 to 2048 entries
// and go through each run in the order of the rows: what an expert gets from the run lies together.  A run's tokens
// (2 MiB at 8 choices and 8 KiB) stay in the L2 of the one XCD that takes the run, so reading a token once per row costs no
// memory traffic.  The order inside a bucket of rows is whatever the counters give: it has no part in any result.
constexpr uint32_t kOrderMaxRun = 2048;
constexpr uint32_t kOrderBuckets = 1024;        // buckets of 1 << shift rows, and one more for entries without a row
constexpr int kOrderBlock = 1024;
struct OrderedEntry {
    int32_t row;                // -1: none
    uint32_t entry;
};

__global__ void __launch_bounds__(kOrderBlock)
token_order_kernel(const int32_t* positions, uint64_t n, uint32_t run, uint64_t rows, uint32_t shift, OrderedEntry* order) {
    __shared__ uint32_t slot[kOrderBuckets + 1];
    __shared__ uint32_t wave_end[kOrderBlock / 64];
    static_assert(kOrderBuckets == kOrderBlock && kOrderMaxRun == 2 * kOrderBlock, "a bucket and at most two entries per lane");
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint64_t first = (uint64_t)blockIdx.x * run;
    const uint64_t end = first + run < n ? first + run : n;
    slot[tid] = 0;
    if (tid == 0) slot[kOrderBuckets] = 0;
    __syncthreads();
    int32_t p[2];
    uint32_t bucket[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const uint64_t i = first + tid + (uint64_t)u * kOrderBlock;
        p[u] = i < end ? positions[i] : -1;
        if (p[u] >= 0 && (uint64_t)p[u] >= rows) p[u] = -1;
        bucket[u] = p[u] < 0 ? kOrderBuckets : (uint32_t)p[u] >> shift;
        if (i < end) atomicAdd(&slot[bucket[u]], 1u);
    }
    __syncthreads();
    const uint32_t mine = slot[tid];
    uint32_t incl = mine;
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint32_t up = __shfl_up(incl, d, 64);
        if (lane >= d) incl += up;
    }
    if (lane == 63) wave_end[wave] = incl;
    __syncthreads();
    uint32_t base = 0;
    for (uint32_t w = 0; w < wave; w++) base += wave_end[w];
    slot[tid] = base + incl - mine;
    if (tid == kOrderBlock - 1) slot[kOrderBuckets] = base + incl;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const uint64_t i = first + tid + (uint64_t)u * kOrderBlock;
        if (i < end) order[first + atomicAdd(&slot[bucket[u]], 1u)] = OrderedEntry{ p[u], (uint32_t)i };
    }
}

// A block takes one entry, or, MULTI, an entry per group of 1 << log_lanes lanes: whole waves, so that all that follows from the
// entry is on the scalar unit (as the lanes' own values it cost a tenth).  Entries come run after run, eight runs side by
// side, one per XCD (blocks go round the XCDs by their index).
constexpr int kOrderedBlock = 512;         // lanes at most
constexpr uint32_t kOrderedMultiBlock = 256;
template <bool MULTI>
struct OrderedLane {
    uint64_t at;                // the group's place in the order
    uint32_t lanes, lane;
    __device__ __forceinline__ OrderedLane(uint32_t block, uint32_t log_lanes, uint32_t log_run) {
        lanes = MULTI ? 1u << log_lanes : blockDim.x;
        lane = MULTI ? threadIdx.x & (lanes - 1) : threadIdx.x;
        const uint32_t xcd = block & 7u;
        const uint32_t r = MULTI ? (block >> 3) * (kOrderedMultiBlock >> log_lanes) + __builtin_amdgcn_readfirstlane(threadIdx.x >> log_lanes) : block >> 3;
        at = ((((uint64_t)(r >> log_run) << 3) + xcd) << log_run) + (r & ((1u << log_run) - 1));
    }
};

// A group of lanes copies one entry's row.
template <class E, bool MULTI>
__global__ void __launch_bounds__(kOrderedBlock)
token_dispatch_ordered_kernel(const unsigned char* x, uint64_t ldx, uint32_t nvec, uint32_t tail, uint32_t top_k, uint64_t n, uint32_t experts,
                              const OrderedEntry* order, uint32_t log_lanes, uint32_t log_run, const int32_t* counts, const int32_t* offsets,
                              unsigned char* out, uint64_t ldo, uint64_t rows) {
    constexpr uint32_t VEC = 16 / sizeof(E);
    const uint32_t pads = pad_blocks(experts);
    if (blockIdx.x < pads) {
        clear_padding<E>(blockIdx.x, experts, counts, offsets, rows, out, ldo, nvec, tail);
        return;
    }
    const OrderedLane<MULTI> my(blockIdx.x - pads, log_lanes, log_run);
    if (my.at >= n) return;
    const OrderedEntry e = order[my.at];
    if (e.row < 0) return;
    const uint32_t lane = my.lane;
    const unsigned char* src = x + (uint64_t)(e.entry / top_k) * ldx * sizeof(E);
    unsigned char* o = out + (uint64_t)e.row * ldo * sizeof(E);
    for (uint32_t v = lane; v < nvec; v += my.lanes) st_loose((u32x4_u*)o + v, ((const u32x4_u*)src)[v]);
    if (lane < tail) st_elem<E>(o, (uint64_t)nvec * VEC + lane, ld_elem<E>(src, (uint64_t)nvec * VEC + lane));
}

// A group of lanes takes one entry: its row's gradient and, with DOT, its weight's.  The dot product is summed lane by lane over
// the columns, then over the wave and the group's waves in a fixed order.
template <class V, bool DOT, bool MULTI>
__global__ void __launch_bounds__(kOrderedBlock)
token_backward_ordered_kernel(const unsigned char* grad, uint64_t ldg, const unsigned char* y, uint64_t ldy, uint32_t nvec, uint32_t tail,
                              uint32_t top_k, uint64_t n, uint32_t experts, const OrderedEntry* order, uint32_t log_lanes, uint32_t log_run,
                              const float* weights, const int32_t* counts, const int32_t* offsets, unsigned char* grad_y, uint64_t ldd,
                              uint64_t rows, float* grad_weights) {
    typedef typename V::elem_t E;
    constexpr int VEC = V::VEC;
    const uint32_t pads = pad_blocks(experts);
    if (blockIdx.x < pads) {
        clear_padding<E>(blockIdx.x, experts, counts, offsets, rows, grad_y, ldd, nvec, tail);
        return;
    }
    __shared__ float part[kOrderedBlock / 64];
    const OrderedLane<MULTI> my(blockIdx.x - pads, log_lanes, log_run);
    const uint32_t lane = my.lane;
    OrderedEntry e = { -1, 0 };
    if (my.at < n) e = order[my.at];
    float dot = 0.0f;
    if (e.row >= 0) {
        const float f = weights ? weights[e.entry] : 1.0f;
        const unsigned char* g = grad + (uint64_t)(e.entry / top_k) * ldg * sizeof(E);
        const unsigned char* r = DOT ? y + (uint64_t)e.row * ldy * sizeof(E) : nullptr;
        unsigned char* d = grad_y + (uint64_t)e.row * ldd * sizeof(E);
        for (uint32_t v = lane; v < nvec; v += my.lanes) {
            u32x4 b;
            if (DOT) b = ld_loose((const u32x4_u*)r + v);
            float a[VEC], c[VEC];
            V::widen(((const u32x4_u*)g)[v], a);
#pragma unroll
            for (int i = 0; i < VEC; i++) c[i] = f * a[i];
            st_loose((u32x4_u*)d + v, V::narrow(c));
            if (DOT) {
                V::widen(b, c);
#pragma unroll
                for (int i = 0; i < VEC; i++) dot = __builtin_fmaf(a[i], c[i], dot);
            }
        }
        if (lane < tail) {
            const uint64_t i = (uint64_t)nvec * VEC + lane;
            const float a = V::widen1(ld_elem<E>(g, i));
            st_elem<E>(d, i, V::narrow1(f * a));
            if (DOT) dot = __builtin_fmaf(a, V::widen1(ld_elem<E>(r, i)), dot);
        }
    }
    if (DOT) {
        dot = wave_sum(dot);
        if ((threadIdx.x & 63u) == 0) part[threadIdx.x >> 6] = dot;
        __syncthreads();
        if (lane == 0 && my.at < n) {
            float sum = 0.0f;
            for (uint32_t q = 0; q < my.lanes / 64; q++) sum += part[(threadIdx.x >> 6) + q];
            grad_weights[e.entry] = sum;            // 0 for an entry without a row
        }
    }
}

// ---- token by token -----------------------------------------------------------------------------------------------------------

// A token's columns are read once and stored to its rows.
template <class E, int U>
__global__ void __launch_bounds__(kBlock)
token_dispatch_kernel(const unsigned char* x, uint64_t ldx, RowShape s, uint32_t experts, const int32_t* positions, const int32_t* counts,
                      const int32_t* offsets, unsigned char* out, uint64_t ldo, uint64_t rows) {
    constexpr uint32_t VEC = 16 / sizeof(E);
    const uint32_t pads = pad_blocks(experts);
    if (blockIdx.y < pads) {
        if (blockIdx.x == 0) clear_padding<E>(blockIdx.y, experts, counts, offsets, rows, out, ldo, s.nvec, s.tail);
        return;
    }
    const uint32_t token_block = blockIdx.y - pads, token_blocks = gridDim.y - pads;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t per_block = (kBlock / 64) >> s.log_waves, width = 64u << s.log_waves;
    const uint32_t col = (wave & ((1u << s.log_waves) - 1)) * 64u + lane;
    for (uint64_t t = (uint64_t)token_block * per_block + (wave >> s.log_waves); t < s.tokens; t += (uint64_t)token_blocks * per_block) {
        const unsigned char* src = x + t * ldx * sizeof(E);
        const int32_t* pos = positions + t * s.top_k;
        for (uint32_t c = blockIdx.x; c < s.cols; c += gridDim.x) {
            const uint32_t v0 = c * width * U + col;
            u32x4 v[U];
#pragma unroll
            for (int u = 0; u < U; u++)
                if (v0 + width * u < s.nvec) v[u] = ld_loose((const u32x4_u*)src + v0 + width * u);
            const bool edge = c == s.cols - 1 && col < s.tail;
            E one = 0;
            if (edge) one = ld_elem<E>(src, (uint64_t)s.nvec * VEC + col);
            for (uint32_t j = 0; j < s.top_k; j++) {
                const int32_t p = pos[j];
                if (p < 0 || (uint64_t)p >= rows) continue;
                unsigned char* o = out + (uint64_t)p * ldo * sizeof(E);
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (v0 + width * u < s.nvec) st_loose((u32x4_u*)o + v0 + width * u, v[u]);
                if (edge) st_elem<E>(o, (uint64_t)s.nvec * VEC + col, one);
            }
        }
    }
}

// The sum runs over the entries in order, in fp32 with one fused multiply-add each, and is rounded once.
template <class V, int U, int K>
__global__ void __launch_bounds__(kBlock)
token_combine_kernel(const unsigned char* y, uint64_t ldy, uint64_t rows, RowShape s, const int32_t* positions, const float* weights,
                     unsigned char* out, uint64_t ldo) {
    typedef typename V::elem_t E;
    constexpr int VEC = V::VEC;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t per_block = (kBlock / 64) >> s.log_waves, width = 64u << s.log_waves;
    const uint32_t col = (wave & ((1u << s.log_waves) - 1)) * 64u + lane;
    for (uint64_t t = (uint64_t)blockIdx.y * per_block + (wave >> s.log_waves); t < s.tokens; t += (uint64_t)gridDim.y * per_block) {
        unsigned char* o = out + t * ldo * sizeof(E);
        for (uint32_t c = blockIdx.x; c < s.cols; c += gridDim.x) {
            const uint32_t v0 = c * width * U + col;
            const bool edge = c == s.cols - 1 && col < s.tail;
            float acc[U][VEC] = {}, one = 0.0f;
            for (uint32_t j0 = 0; j0 < s.top_k; j0 += K) {
                const uint32_t k = s.top_k - j0 < (uint32_t)K ? s.top_k - j0 : (uint32_t)K;
                int32_t p[K];
                load_positions<K>(positions + t * s.top_k + j0, k, rows, p);
                const float* w = weights ? weights + t * s.top_k + j0 : nullptr;
                u32x4 x[U][K];
                E e[K];
#pragma unroll
                for (int j = 0; j < K; j++) {
                    if (p[j] < 0) continue;
                    const unsigned char* src = y + (uint64_t)p[j] * ldy * sizeof(E);
#pragma unroll
                    for (int u = 0; u < U; u++)
                        if (v0 + width * u < s.nvec) x[u][j] = ld_loose((const u32x4_u*)src + v0 + width * u);
                    if (edge) e[j] = ld_elem<E>(src, (uint64_t)s.nvec * VEC + col);
                }
#pragma unroll
                for (int j = 0; j < K; j++) {
                    if (p[j] < 0) continue;
                    const float f = w ? w[j] : 1.0f;
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        float g[VEC];
                        V::widen(x[u][j], g);
#pragma unroll
                        for (int i = 0; i < VEC; i++) acc[u][i] = __builtin_fmaf(f, g[i], acc[u][i]);
                    }
                    if (edge) one = __builtin_fmaf(f, V::widen1(e[j]), one);
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++)
                if (v0 + width * u < s.nvec) st_loose((u32x4_u*)o + v0 + width * u, V::narrow(acc[u]));
            if (edge) st_elem<E>(o, (uint64_t)s.nvec * VEC + col, V::narrow1(one));
        }
    }
}

// A block takes one token: a vector of its gradient row is read once and meets the rows of up to K entries.  The dot products
// are summed in fp32, lane by lane over the columns, then over the wave and the block in a fixed order.
template <class V, int K, bool DOT>
__global__ void __launch_bounds__(1024)
token_combine_backward_kernel(const unsigned char* grad, uint64_t ldg, const unsigned char* y, uint64_t ldy, uint64_t rows, RowShape s,
                              uint32_t experts, const int32_t* positions, const float* weights, const int32_t* counts,
                              const int32_t* offsets, unsigned char* grad_y, uint64_t ldd, float* grad_weights) {
    typedef typename V::elem_t E;
    constexpr int VEC = V::VEC;
    const uint32_t pads = pad_blocks(experts);
    if (blockIdx.x < pads) {
        clear_padding<E>(blockIdx.x, experts, counts, offsets, rows, grad_y, ldd, s.nvec, s.tail);
        return;
    }
    __shared__ float part[16][K];
    const uint32_t tid = threadIdx.x;
    for (uint64_t t = blockIdx.x - pads; t < s.tokens; t += gridDim.x - pads) {
        const unsigned char* g = grad + t * ldg * sizeof(E);
        for (uint32_t j0 = 0; j0 < s.top_k; j0 += K) {
            const uint32_t k = s.top_k - j0 < (uint32_t)K ? s.top_k - j0 : (uint32_t)K;
            const float* w = weights ? weights + t * s.top_k + j0 : nullptr;
            int32_t p[K];
            load_positions<K>(positions + t * s.top_k + j0, k, rows, p);
            float f[K], dot[K];
#pragma unroll
            for (int j = 0; j < K; j++) {
                f[j] = (uint32_t)j < k && w ? w[j] : 1.0f;
                dot[j] = 0.0f;
            }
            for (uint32_t v = tid; v < s.nvec; v += blockDim.x) {
                u32x4 row[K];
                if (DOT) {
#pragma unroll
                    for (int j = 0; j < K; j++)
                        if (p[j] >= 0) row[j] = ld_loose((const u32x4_u*)(y + (uint64_t)p[j] * ldy * sizeof(E)) + v);
                }
                float a[VEC];
                V::widen(ld_loose((const u32x4_u*)g + v), a);
#pragma unroll
                for (int j = 0; j < K; j++) {
                    if (p[j] < 0) continue;
                    float d[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; i++) d[i] = f[j] * a[i];
                    st_loose((u32x4_u*)(grad_y + (uint64_t)p[j] * ldd * sizeof(E)) + v, V::narrow(d));
                    if (DOT) {
                        float b[VEC];
                        V::widen(row[j], b);
#pragma unroll
                        for (int i = 0; i < VEC; i++) dot[j] = __builtin_fmaf(a[i], b[i], dot[j]);
                    }
                }
            }
            if (tid < s.tail) {
                const uint64_t i = (uint64_t)s.nvec * VEC + tid;
                const float a = V::widen1(ld_elem<E>(g, i));
#pragma unroll
                for (int j = 0; j < K; j++) {
                    if (p[j] < 0) continue;
                    st_elem<E>(grad_y + (uint64_t)p[j] * ldd * sizeof(E), i, V::narrow1(f[j] * a));
                    if (DOT) dot[j] = __builtin_fmaf(a, V::widen1(ld_elem<E>(y + (uint64_t)p[j] * ldy * sizeof(E), i)), dot[j]);
                }
            }
            if (DOT) {
#pragma unroll
                for (int j = 0; j < K; j++) {
                    const float sum = wave_sum(dot[j]);
                    if ((tid & 63u) == 0) part[tid >> 6][j] = sum;
                }
                __syncthreads();
                if (tid < k) {
                    float sum = 0.0f;
                    for (uint32_t q = 0; q < blockDim.x / 64; q++) sum += part[q][tid];
                    grad_weights[t * s.top_k + j0 + tid] = sum;
                }
                __syncthreads();
            }
        }
    }
}

}  // namespace mi
