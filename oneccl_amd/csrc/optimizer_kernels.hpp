// Operators on the gradients of a fused group: the norm over all tensors with the clip coefficient, the AdamW step, and
// its states in 8 bits.
//
// With g' = c g (c: the clip coefficient, an unscaling, or both), for every element:
//   m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2
//   w = w (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// States and weights live in the plan's layout: element i of tensor t at off[t] / (size of a gradient) + i.
//
// 8-bit states: 256 consecutive elements of a tensor share one power of two per state, 2^(s - 127).
//   m: a sign, 4 bits of exponent and 3 of mantissa (e4m3, largest 448, 0x7f and 0xff NaN)
//   v: 4 bits of exponent and 4 of mantissa, no sign: code c < 16 stands for c, others for (16 + c % 16) 2^(c / 16 - 1);
//      255 is NaN, the largest value 30 * 2^14
// s is the smallest for which the block's largest finite magnitude is representable, at least 1.  A value that is not finite
// (or a v below zero, which no step makes) becomes NaN.  A v above zero never becomes zero (it would be a divisor of the next m), but 1.
// Both formats are pieces of the fp32 format, so a value is coded by a multiplication with a power of two that puts the
// format's smallest normal value on fp32's, and a rounding of the fp32 bits: to nearest even, or by adding random bits.
#pragma once

#include "float_vec.hpp"
#include "fusion_kernels.hpp"

namespace mi {

constexpr uint32_t kStateBlock = MI_CCL_STATE_BLOCK;    // elements of one 8-bit block
constexpr uint32_t kAdamwBlock = 128;                   // lanes of a block of the AdamW step
constexpr uint32_t kAdamwTile = 4 * kAdamwBlock;        // its elements
static_assert(kStateBlock == 64 * 4, "four elements of each lane of a wave are one 8-bit block");

// ---- norm ---------------------------------------------------------------------------------------------------------------
// Partial sums of one launch: three blocks per CU, each with the next item's address at hand.  800 M bf16 elements: 226 us
// with 768 blocks (7.07 TB/s, what reading alone reaches), 250 with 512, 232 with 1,024, 246 with 2,048 to 16,384; 265 where
// the blocks look an item up when they come to it.
constexpr uint32_t kNormBlocks = 768;

struct NormTables {
    const uint64_t* off;
    const uint64_t* bytes;
    const FusionItem* items;
    uint32_t nitems, t0;
};

// What a block needs of an item: fetched while the item before it is summed up, so that the chain from the item to the
// tensor's tables and pointer is off the path of the data.
template <uint32_t ES, bool BUFFER>
struct NormItem {
    const unsigned char* g;
    uint32_t nelem;
    __device__ __forceinline__ NormItem(const FusionPtrs& grads, const unsigned char* buffer, const NormTables& tb, uint32_t it) {
        const FusionItem w = tb.items[it < tb.nitems ? it : tb.nitems - 1];
        const uint64_t lo = (uint64_t)w.c * kFusionChunk, left = tb.bytes[w.t] - lo;
        nelem = (left < kFusionChunk ? (uint32_t)left : kFusionChunk) / ES;
        g = (BUFFER ? buffer + tb.off[w.t] : (const unsigned char*)(uintptr_t)grads.get(w.t - tb.t0)) + lo;
    }
};

// One double per block.  Squares and sums are fp64 throughout, in a fixed order: no finite gradient overflows or is lost, and
// memory is still what bounds the kernel (226 us for 800 M bf16 elements, with squares in fp32 226 too).
template <class V, bool BUFFER>
__global__ void __launch_bounds__(kBlock)
fusion_norm_kernel(FusionPtrs grads, const unsigned char* buffer, NormTables tb, double* partial) {
    typedef typename V::elem_t E;
    constexpr uint32_t ES = sizeof(E), VEC = V::VEC;
    __shared__ double part[kBlock / 64];
    const uint32_t tid = threadIdx.x;
    double sum[2] = { 0.0, 0.0 };
    NormItem<ES, BUFFER> next(grads, buffer, tb, blockIdx.x);
    for (uint32_t it = blockIdx.x; it < tb.nitems; it += gridDim.x) {
        const unsigned char* g = next.g;
        const uint32_t nelem = next.nelem;
        uint32_t head = fusion_head<ES>(g);
        if (head > nelem) head = nelem;
        const uint32_t nvec = (nelem - head) / VEC, tail = nelem - head - nvec * VEC;
        u32x4 x[4];
#pragma unroll
        for (int u = 0; u < 4; u++)
            x[u] = tid + u * kBlock < nvec ? ld_loose((const u32x4_u*)(g + head * ES) + tid + u * kBlock) : u32x4{ 0, 0, 0, 0 };
        float edge = 0.0f;
        if (tid < head + tail) edge = V::widen1(ld_elem<E>(g, tid < head ? tid : head + nvec * VEC + (tid - head)));
        next = NormItem<ES, BUFFER>(grads, buffer, tb, it + gridDim.x);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            float f[VEC];
            V::widen(x[u], f);
#pragma unroll
            for (uint32_t i = 0; i < VEC; i++) sum[i % 2] = __builtin_fma((double)f[i], (double)f[i], sum[i % 2]);
        }
        sum[0] = __builtin_fma((double)edge, (double)edge, sum[0]);
    }
    sum[0] = wave_sum(sum[0] + sum[1]);
    if ((tid & 63u) == 0) part[tid >> 6] = sum[0];
    __syncthreads();
    if (tid == 0) {
        double s = 0.0;
        for (int q = 0; q < kBlock / 64; q++) s += part[q];
        partial[blockIdx.x] = s;
    }
}

// result[0] = |multiplier| sqrt(sum), result[1] = multiplier * min(1, max_norm / (result[0] + 1e-6)) (max_norm <= 0: multiplier);
// NaN where the norm is not finite, which the AdamW step takes as "leave everything as it is".
__global__ void __launch_bounds__(1024)
fusion_norm_finish_kernel(const double* partial, uint32_t n, double multiplier, double max_norm, float* result) {
    __shared__ double part[16];
    const uint32_t tid = threadIdx.x;
    double sum = 0.0;
    for (uint32_t i = tid; i < n; i += 1024) sum += partial[i];
    sum = wave_sum(sum);
    if ((tid & 63u) == 0) part[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) {
        double s = 0.0;
        for (int q = 0; q < 16; q++) s += part[q];
        const float norm = (float)(fabs(multiplier) * sqrt(s));
        double coef = multiplier;
        if (max_norm > 0.0) {
            const double c = max_norm / ((double)norm + 1e-6);
            if (c < 1.0) coef *= c;
        }
        result[0] = norm;
        result[1] = __builtin_isfinite(norm) ? (float)coef : __builtin_nanf("");
    }
}

// ---- 8-bit states -------------------------------------------------------------------------------------------------------

// The largest of a number over the wave (which holds one block), the same in every lane: within rows of 16 lanes with
// DPP, whose exchange is part of the max instruction, across the four rows on the scalar unit: no trip through the LDS crossbar.
template <int CTRL>
__device__ __forceinline__ uint32_t max_across(uint32_t x) {
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false);
    return x > y ? x : y;
}
__device__ __forceinline__ uint32_t block_max(uint32_t x) {
    x = max_across<0xb1>(x);        // quad_perm [1, 0, 3, 2]
    x = max_across<0x4e>(x);        // quad_perm [2, 3, 0, 1]
    x = max_across<0x141>(x);       // row_half_mirror
    x = max_across<0x140>(x);       // row_mirror
    const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)x, 0), b = (uint32_t)__builtin_amdgcn_readlane((int)x, 16);
    const uint32_t c = (uint32_t)__builtin_amdgcn_readlane((int)x, 32), d = (uint32_t)__builtin_amdgcn_readlane((int)x, 48);
    const uint32_t ab = a > b ? a : b, cd = c > d ? c : d;
    return ab > cd ? ab : cd;
}
constexpr uint32_t kInfBits = 0x7f800000u;
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return as_u32(x) & 0x7fffffffu; }

// the byte s for a block whose largest magnitude has these bits: TOP and MANT say that the format's largest value is
// 2^TOP * (1 + MANT / 2^23)
template <uint32_t TOP, uint32_t MANT>
__device__ __forceinline__ uint32_t state_scale(uint32_t b) {
    const int s = (int)(b >> 23) - (int)TOP + ((b & 0x7fffffu) > MANT ? 1 : 0);
    return s < 1 ? 1u : (uint32_t)s;
}
__device__ __forceinline__ uint32_t scale_avg(uint32_t largest) { return state_scale<8, 0x600000>(largest); }    // 448
__device__ __forceinline__ uint32_t scale_sq(uint32_t largest) { return state_scale<18, 0x700000>(largest); }    // 30 * 2^14

// fp32 bits to a code of SHIFT bits less: nearest even, or up with the probability of what is cut off (16 random bits)
template <int SHIFT, bool RANDOM>
__device__ __forceinline__ uint32_t round_bits(uint32_t b, uint32_t random16) {
    if (RANDOM) return (b + (random16 << (SHIFT - 16))) >> SHIFT;
    return (b + ((1u << (SHIFT - 1)) - 1) + ((b >> SHIFT) & 1u)) >> SHIFT;
}
// The codes of finite values (a v not below zero); code_* of CHECKED any others too.
template <bool RANDOM, bool CHECKED>
__device__ __forceinline__ uint32_t code_avg(float m, uint32_t s, uint32_t random16) {
    uint32_t c = round_bits<20, RANDOM>(as_u32(__builtin_ldexpf(fabsf(m), 7 - (int)s)), random16);
    if (CHECKED && magnitude_bits(m) >= kInfBits) c = 0x7fu;
    return c | ((as_u32(m) >> 24) & 0x80u);
}
template <bool RANDOM, bool CHECKED>
__device__ __forceinline__ uint32_t code_sq(float v, uint32_t s, uint32_t random16) {
    uint32_t c = round_bits<19, RANDOM>(as_u32(__builtin_ldexpf(fabsf(v), -3 - (int)s)), random16);
    const uint32_t least = as_u32(v) < 1u ? as_u32(v) : 1u;         // 1 for what is above zero
    c = c > least ? c : least;
    if (CHECKED) c = v >= 0.0f && v < __builtin_inff() ? (v == 0.0f ? 0u : c) : 255u;
    return c;
}
// Four codes of one block; v_cvt_pk_f32_fp8 and v_cvt_pk_fp8_f32 are this format's own conversions (to nearest even).
__device__ __forceinline__ void decode4(uint32_t cm, uint32_t cv, uint32_t sm, uint32_t sv, float* m, float* v) {
    const float unit = as_f32(sm << 23);
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)cm, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)cm, true);
    m[0] = lo[0] * unit;
    m[1] = lo[1] * unit;
    m[2] = hi[0] * unit;
    m[3] = hi[1] * unit;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = __builtin_ldexpf(as_f32(((cv >> (8 * i)) & 0xffu) << 19), (int)sv + 3);
    if ((~cv - 0x01010101u) & cv & 0x80808080u) {                   // a byte of 255 among them (or a false alarm next to one)
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (((cv >> (8 * i)) & 0xffu) == 255u) v[i] = __builtin_nanf("");
    }
}
struct Coded {
    uint32_t cm, cv;            // four codes each
    uint32_t sm, sv;            // the block's scales
};

// 32 random bits of an element: a multiply-and-shift mix of its index in the layout (the low half; the high half goes into the
// key) and the step's key.
__device__ __host__ __forceinline__ uint32_t mix32(uint32_t x) {
    x ^= x >> 16;
    x *= 0x9E3779B1u;
    x ^= x >> 15;
    x *= 0x85EBCA77u;
    return x ^ (x >> 16);
}
__device__ __host__ __forceinline__ uint32_t step_key(uint64_t seed, uint64_t step) {
    return mix32(mix32((uint32_t)seed + (uint32_t)step * 0x9E3779B1u) ^ (uint32_t)(seed >> 32));
}
// Four elements of every lane of a wave, one block in all, coded; index: of the lane's first (a multiple of 4), for its random
// bits.  A block with anything that is not finite (or a negative v) goes the long way, the whole wave together.
template <bool RANDOM, bool CHECKED>
__device__ __forceinline__ void code4(const float* m, const float* v, uint32_t at, uint32_t key, Coded& c) {
    if (!RANDOM && !CHECKED) {
        const float unit = as_f32((254u - c.sm) << 23);
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(m[0] * unit, m[1] * unit, 0, false);
        c.cm = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(m[2] * unit, m[3] * unit, w, true);
    }
    else
        c.cm = 0;
    c.cv = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t r = RANDOM ? mix32(at ^ (uint32_t)i ^ key) : 0;
        if (RANDOM || CHECKED) c.cm |= code_avg<RANDOM, CHECKED>(m[i], c.sm, r & 0xffffu) << (8 * i);
        c.cv |= code_sq<RANDOM, CHECKED>(v[i], c.sv, r >> 16) << (8 * i);
    }
}
template <bool RANDOM>
__device__ __forceinline__ Coded encode4(const float* m, const float* v, uint64_t index, uint32_t key) {
    uint32_t bm = 0, bv = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t a = magnitude_bits(m[i]), b = as_u32(v[i]);
        bm = bm > a ? bm : a;
        bv = bv > b ? bv : b;
    }
    bm = block_max(bm);
    bv = block_max(bv);                 // a sign bit makes it the largest
    const uint32_t at = (uint32_t)index, k = key ^ ((uint32_t)(index >> 32) * 0x85EBCA77u);
    Coded c;
    if (bm < kInfBits && bv < kInfBits) {
        c.sm = scale_avg(bm);
        c.sv = scale_sq(bv);
        code4<RANDOM, false>(m, v, at, k, c);
    }
    else {
        bm = bv = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t a = magnitude_bits(m[i]), b = magnitude_bits(v[i]);
            if (a < kInfBits && a > bm) bm = a;
            if (b < kInfBits && b > bv) bv = b;
        }
        c.sm = scale_avg(block_max(bm));
        c.sv = scale_sq(block_max(bv));
        code4<RANDOM, true>(m, v, at, k, c);
    }
    return c;
}

// ---- a lane's elements ----------------------------------------------------------------------------------------------------

// Four elements of consecutive memory, as many bytes as their type needs (16, 8 or 4): with lane after lane behind each other
// every access of a wave covers one unbroken run, whatever the widths of the arrays that meet in one element are.
typedef u32x2 u32x2_u __attribute__((aligned(1)));
typedef uint32_t u32_u __attribute__((aligned(1)));

// WHOLE: all four, else elements [from, to) of them (none when from >= to).
struct Span {
    int from, to;
    __device__ __forceinline__ bool has(int i) const { return i >= from && i < to; }
    __device__ __forceinline__ bool whole() const { return from <= 0 && to >= 4; }
};
template <class V, bool WHOLE>
__device__ __forceinline__ void load4(const void* p, Span n, float* f) {
    typedef typename V::elem_t E;
    if (WHOLE || n.whole()) {
        if (sizeof(E) == 4) V::widen(ld_loose((const u32x4_u*)p), f);
        else V::widen_half(__builtin_nontemporal_load((const u32x2_u*)p), f);
    }
    else {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = n.has(i) ? V::widen1(ld_elem<E>(p, i)) : 0.0f;
    }
}
template <class V, bool WHOLE>
__device__ __forceinline__ void store4(void* p, Span n, const float* f) {
    typedef typename V::elem_t E;
    if (WHOLE || n.whole()) {
        if (sizeof(E) == 4) st_loose((u32x4_u*)p, V::narrow(f));
        else __builtin_nontemporal_store(V::narrow_half(f), (u32x2_u*)p);
    }
    else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (n.has(i)) st_elem<E>(p, i, V::narrow1(f[i]));
    }
}
template <bool WHOLE>
__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, Span n) {
    if (WHOLE || n.whole()) return __builtin_nontemporal_load((const u32_u*)p);
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (n.has(i)) c |= (uint32_t)p[i] << (8 * i);
    return c;
}
template <bool WHOLE>
__device__ __forceinline__ void store_codes(uint8_t* p, Span n, uint32_t c) {
    if (WHOLE || n.whole()) {
        __builtin_nontemporal_store(c, (u32_u*)p);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (n.has(i)) p[i] = (uint8_t)(c >> (8 * i));
}

// ---- AdamW --------------------------------------------------------------------------------------------------------------

// What follows from the learning rate and the step's number.
struct AdamwDerived {
    float decay;            // 1 - lr wd
    float step_size;        // lr / (1 - beta1^t)
    float root_scale;       // 1 / sqrt(1 - beta2^t)
    uint32_t key;           // of the step's random bits
};
static_assert(sizeof(AdamwDerived) == MI_CCL_ADAMW_WORKSPACE, "the header says how much memory it takes");
struct AdamwHyper {
    double lr, weight_decay, beta1, beta2;
    int64_t step;
    uint64_t seed;
};
struct AdamwScalars {
    float beta1, rest1, beta2, rest2, eps;
    AdamwDerived d;
    const AdamwDerived* derived;    // or NULL: in memory, from numbers that the host does not know
    const float* grad_scale;
};

// b^t by squaring, in fp64
__host__ __device__ inline double whole_power(double b, int64_t t) {
    double r = 1.0;
    for (; t > 0; t >>= 1) {
        if (t & 1) r *= b;
        b *= b;
    }
    return r;
}
__host__ __device__ inline AdamwDerived adamw_derive(const AdamwHyper& h) {
    AdamwDerived d;
    d.decay = (float)(1.0 - h.lr * h.weight_decay);
    d.step_size = (float)(h.lr / (1.0 - whole_power(h.beta1, h.step)));
    d.root_scale = (float)(1.0 / sqrt(1.0 - whole_power(h.beta2, h.step)));
    d.key = step_key(h.seed, (uint64_t)h.step);
    return d;
}
// A launch of its own: the some 200 fp64 instructions in every wave of the step would make it a third slower (130 M parameters with
// 8-bit states 471 against 337 us).
__global__ void adamw_derive_kernel(AdamwHyper h, const float* lr, const int64_t* step, AdamwDerived* out) {
    if (lr) h.lr = (double)*lr;
    if (step) h.step = *step;
    *out = adamw_derive(h);
}

struct AdamwTables {
    const uint64_t* off;            // bytes of gradients
    const uint64_t* bytes;
    const FusionItem* items;
    uint32_t t0;
    uint32_t log_esize;             // of a gradient
};
struct AdamwState {
    void* avg;
    void* sq;
    uint8_t* scales;                // 8 bits: two bytes of every block
    float* master;
};

// sqrt to one ulp: v_sqrt_f32, whose argument may not be denormal, hence the detour for the smallest; `scale` is a factor of
// the result.
__device__ __forceinline__ float scaled_sqrt(float v, float scale) {
    const bool tiny = v < 0x1p-96f;
    return __builtin_amdgcn_sqrtf(v * (tiny ? 0x1p64f : 1.0f)) * (tiny ? scale * 0x1p-32f : scale);
}
// One element's step: m, v and x (the weight) in, out.
__device__ __forceinline__ void adamw_element(const AdamwScalars& a, float g, float& m, float& v, float& x) {
    m = m * a.beta1 + g * a.rest1;
    v = v * a.beta2 + (g * g) * a.rest2;
    const float root = scaled_sqrt(v, a.d.root_scale) + a.eps;
    x = x * a.d.decay - (m * __builtin_amdgcn_rcpf(root)) * a.d.step_size;
}

// A tensor's arrays, each at the tensor's element 0.
struct AdamwTensor {
    unsigned char* p;
    const unsigned char* g;
    float* master;
    void* avg;
    void* sq;
    uint8_t* scales;
    uint64_t at;                // element 0 in the plan's layout
    int64_t count;
};

enum { STATE_FP32 = 0, STATE_NEAREST = 1, STATE_RANDOM = 2 };

// Elements [e0, e0 + kAdamwTile) of a tensor, those that it has (WHOLE: all of them), four in a row of every lane: one 8-bit
// block is what a wave has, and every access of a wave is one unbroken run.
template <class P, class G, bool MASTER, int STATE, bool WHOLE>
__device__ __forceinline__ void adamw_tile(const AdamwTensor& t, int64_t e0, const AdamwScalars& a, float scale) {
    constexpr int64_t GS = sizeof(typename G::elem_t), PS = sizeof(typename P::elem_t);
    const uint32_t e = threadIdx.x * 4;
    Span n = { 0, 4 };                                          // what the lane has of its four
    if (!WHOLE) {
        const int64_t lo = -(e0 + e), hi = t.count - (e0 + e);
        n.from = lo > 4 ? 4 : lo < 0 ? 0 : (int)lo;
        n.to = hi > 4 ? 4 : hi < 0 ? 0 : (int)hi;
        if (n.from >= n.to) n = Span{ 4, 0 };
    }
    unsigned char* const p = t.p + e0 * PS;
    float* const master = t.master + e0;
    float* const avg = (float*)t.avg + e0;
    float* const sq = (float*)t.sq + e0;
    uint8_t* const avg8 = (uint8_t*)t.avg + e0;
    uint8_t* const sq8 = (uint8_t*)t.sq + e0;
    uint8_t* const scales = t.scales + 2 * (e0 / kStateBlock + threadIdx.x / 64);
    float g[4], m[4], v[4], x[4];
    load4<G, WHOLE>(t.g + e0 * GS + e * GS, n, g);
    if (MASTER) load4<F32Vec, WHOLE>(master + e, n, x);
    else load4<P, WHOLE>(p + e * PS, n, x);
    if (STATE == STATE_FP32) {
        load4<F32Vec, WHOLE>(avg + e, n, m);
        load4<F32Vec, WHOLE>(sq + e, n, v);
    }
    else {
        const uint32_t cm = load_codes<WHOLE>(avg8 + e, n), cv = load_codes<WHOLE>(sq8 + e, n);
        uint32_t sm = 0, sv = 0;
        if (WHOLE || n.to) {
            sm = scales[0];
            sv = scales[1];
        }
        decode4(cm, cv, sm, sv, m, v);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) adamw_element(a, g[i] * scale, m[i], v[i], x[i]);
    if (MASTER) store4<F32Vec, WHOLE>(master + e, n, x);
    store4<P, WHOLE>(p + e * PS, n, x);
    if (STATE == STATE_FP32) {
        store4<F32Vec, WHOLE>(avg + e, n, m);
        store4<F32Vec, WHOLE>(sq + e, n, v);
    }
    else {
        if (!WHOLE) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (!n.has(i)) m[i] = v[i] = 0.0f;              // no part of the block
        }
        const Coded c = encode4<STATE == STATE_RANDOM>(m, v, t.at + e0 + e, a.d.key);
        store_codes<WHOLE>(avg8 + e, n, c.cm);
        store_codes<WHOLE>(sq8 + e, n, c.cv);
        if ((WHOLE || n.to) && (threadIdx.x & 63u) == 0) {
            scales[0] = (uint8_t)c.sm;
            scales[1] = (uint8_t)c.sv;
        }
    }
}

// A block of threads takes kAdamwTile elements of a tensor.  What bounds the step is memory: 28 bytes per parameter with
// 32-bit states, 16 with 8-bit ones and an fp32 copy of the weights, in four arrays read and four written, which a bare loop
// over such arrays moves at 5.9 to 6.1 TB/s.  Small tiles, read once and written once, are what comes nearest: 200 M parameters
// with 32-bit states, tight layout, 960 us (5.83 TB/s) with 512 elements, 998 with 1,024, 1,018 with 2,048; 130 M with 8-bit states
// 337 us (6.18 TB/s), 348 with two groups of four per lane.
// With 32-bit states in a tight layout a tensor may start anywhere in its arrays.  The tiles are cut where the states cross a
// 256-byte boundary, `back` elements before the multiples of kAdamwTile, so that no two blocks write to one line; tile 0 has
// `back` elements less, and the tensor's last block takes a second, short tile when that leaves elements over.
template <class P, class G, bool MASTER, int STATE>
__global__ void __launch_bounds__(kAdamwBlock)
fusion_adamw_kernel(FusionPtrs params, FusionPtrs grads, const unsigned char* buffer, AdamwTables tb, AdamwState st, AdamwScalars a) {
    constexpr uint32_t GS = sizeof(typename G::elem_t);
    constexpr uint32_t kItemElems = kFusionChunk / GS, kSubs = kItemElems / kAdamwTile;
    float scale = 1.0f;
    if (a.grad_scale) {
        scale = *a.grad_scale;
        if (!(fabsf(scale) < __builtin_inff())) return;         // gradients that are not finite: no step
    }
    if (a.derived) a.d = *a.derived;
    const FusionItem w = tb.items[blockIdx.x / kSubs];
    const uint64_t tile = (uint64_t)w.c * kSubs + blockIdx.x % kSubs, off = tb.off[w.t];
    AdamwTensor t;
    t.count = (int64_t)(tb.bytes[w.t] / GS);
    if (tile * kAdamwTile >= (uint64_t)t.count) return;
    t.at = off / GS;
    t.p = (unsigned char*)(uintptr_t)params.get(w.t - tb.t0);
    t.g = buffer ? buffer + off : (const unsigned char*)(uintptr_t)grads.get(w.t - tb.t0);
    t.master = st.master + t.at;
    t.avg = STATE == STATE_FP32 ? (void*)((float*)st.avg + t.at) : (void*)((uint8_t*)st.avg + t.at);
    t.sq = STATE == STATE_FP32 ? (void*)((float*)st.sq + t.at) : (void*)((uint8_t*)st.sq + t.at);
    t.scales = st.scales + 2 * (t.at / kStateBlock);
    const int64_t back = STATE == STATE_FP32 ? (int64_t)((uintptr_t)t.avg / sizeof(float) % 64) : 0;
    int64_t e0 = (int64_t)(tile * kAdamwTile) - back;
    if (e0 >= 0 && e0 + (int64_t)kAdamwTile <= t.count) adamw_tile<P, G, MASTER, STATE, true>(t, e0, a, scale);
    else adamw_tile<P, G, MASTER, STATE, false>(t, e0, a, scale);
    // the last of the tensor's tiles (there are ceil(count / kAdamwTile)) and elements behind it
    e0 += kAdamwTile;
    if (STATE == STATE_FP32 && e0 < t.count && e0 + back >= t.count) adamw_tile<P, G, MASTER, STATE, false>(t, e0, a, scale);
}

// ---- 8-bit states in and out ----------------------------------------------------------------------------------------------

// The part of an item that a block of the two kernels below takes: G groups of four elements of a lane, a wave 256 G in a row.
constexpr uint32_t kEncodeGroups = 1, kDecodeGroups = 2;
template <uint32_t G>
struct StateTile {
    uint64_t at;        // the lane's first element in the plan's layout; its next group is 256 elements on
    Span n[G];
};
template <uint32_t G>
__device__ __forceinline__ StateTile<G> state_tile(const AdamwTables& tb, uint32_t item_elems) {
    constexpr uint32_t kTile = kBlock * 4 * G;
    const uint32_t subs = item_elems / kTile;
    const FusionItem w = tb.items[blockIdx.x / subs];
    const uint64_t e = (uint64_t)w.c * item_elems + (blockIdx.x % subs) * kTile + (threadIdx.x >> 6) * (256 * G) + (threadIdx.x & 63u) * 4;
    const uint64_t count = tb.bytes[w.t] >> tb.log_esize;
    StateTile<G> s;
    s.at = (tb.off[w.t] >> tb.log_esize) + e;
#pragma unroll
    for (uint32_t q = 0; q < G; q++) {
        const uint64_t f = e + 256 * q;
        s.n[q] = Span{ 0, f >= count ? 0 : count - f < 4 ? (int)(count - f) : 4 };
    }
    return s;
}

// The values of the codes, as fp32 or bfloat16 (which holds every one of them from 2^-126 up).
template <class V>
__global__ void __launch_bounds__(kBlock)
state_decode_kernel(AdamwTables tb, uint32_t item_elems, const uint8_t* avg, const uint8_t* sq, const uint8_t* scales,
                    typename V::elem_t* out_avg, typename V::elem_t* out_sq) {
    constexpr uint32_t G = kDecodeGroups;
    const StateTile<G> t = state_tile<G>(tb, item_elems);
    uint32_t cm[G], cv[G], sm[G], sv[G];
#pragma unroll
    for (uint32_t q = 0; q < G; q++) {
        if (t.n[q].to == 0) continue;
        cm[q] = load_codes<false>(avg + t.at + 256 * q, t.n[q]);
        cv[q] = load_codes<false>(sq + t.at + 256 * q, t.n[q]);
        sm[q] = scales[2 * (t.at / kStateBlock + q)];
        sv[q] = scales[2 * (t.at / kStateBlock + q) + 1];
    }
#pragma unroll
    for (uint32_t q = 0; q < G; q++) {
        if (t.n[q].to == 0) continue;
        float m[4], v[4];
        decode4(cm[q], cv[q], sm[q], sv[q], m, v);
        store4<V, false>(out_avg + t.at + 256 * q, t.n[q], m);
        store4<V, false>(out_sq + t.at + 256 * q, t.n[q], v);
    }
}

// fp32 or bfloat16 values to codes, rounded to nearest.
template <class V>
__global__ void __launch_bounds__(kBlock)
state_encode_kernel(AdamwTables tb, uint32_t item_elems, const typename V::elem_t* in_avg, const typename V::elem_t* in_sq, uint8_t* avg,
                    uint8_t* sq, uint8_t* scales) {
    const StateTile<kEncodeGroups> t = state_tile<kEncodeGroups>(tb, item_elems);
    const Span n = t.n[0];
    float m[4], v[4];
    load4<V, false>(in_avg + t.at, n, m);           // zeros where the tensor has ended: no part of the block
    load4<V, false>(in_sq + t.at, n, v);
    const Coded c = encode4<false>(m, v, t.at, 0);
    store_codes<false>(avg + t.at, n, c.cm);
    store_codes<false>(sq + t.at, n, c.cv);
    if (n.to && (threadIdx.x & 63u) == 0) {
        scales[2 * (t.at / kStateBlock)] = (uint8_t)c.sm;
        scales[2 * (t.at / kStateBlock) + 1] = (uint8_t)c.sv;
    }
}

}  // namespace mi
