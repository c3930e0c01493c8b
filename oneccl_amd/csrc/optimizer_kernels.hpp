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
constexpr uint32_t kLaneElems = 8;                      // elements of one lane
constexpr uint32_t kOptTile = kBlock * kLaneElems;      // elements of one block of threads
static_assert(kOptTile % kStateBlock == 0 && kStateBlock == 32 * kLaneElems, "half a wave holds one 8-bit block");

// ---- norm ---------------------------------------------------------------------------------------------------------------
constexpr uint32_t kNormBlocks = 2048;      // partial sums of one launch

struct NormTables {
    const uint64_t* off;
    const uint64_t* bytes;
    const FusionItem* items;
    uint32_t nitems, t0;
};

// One double per block: squares are summed in fp32 over the at most 33 elements that a lane has of an item (16 KiB of one
// tensor), everything above in fp64 and in a fixed order.
template <class V, bool BUFFER>
__global__ void __launch_bounds__(kBlock)
fusion_norm_kernel(FusionPtrs grads, const unsigned char* buffer, NormTables tb, double* partial) {
    typedef typename V::elem_t E;
    constexpr uint32_t ES = sizeof(E), VEC = V::VEC;
    __shared__ double part[kBlock / 64];
    const uint32_t tid = threadIdx.x;
    double sum = 0.0;
    for (uint32_t it = blockIdx.x; it < tb.nitems; it += gridDim.x) {
        const FusionItem w = tb.items[it];
        const uint64_t lo = (uint64_t)w.c * kFusionChunk, left = tb.bytes[w.t] - lo;
        const uint32_t nelem = (left < kFusionChunk ? (uint32_t)left : kFusionChunk) / ES;
        const unsigned char* g = (BUFFER ? buffer + tb.off[w.t] : (const unsigned char*)(uintptr_t)grads.get(w.t - tb.t0)) + lo;
        uint32_t head = fusion_head<ES>(g);
        if (head > nelem) head = nelem;
        const uint32_t nvec = (nelem - head) / VEC, tail = nelem - head - nvec * VEC;
        float a = 0.0f;
        u32x4 x[4];
#pragma unroll
        for (int u = 0; u < 4; u++)
            x[u] = tid + u * kBlock < nvec ? ld_loose((const u32x4_u*)(g + head * ES) + tid + u * kBlock) : u32x4{ 0, 0, 0, 0 };
#pragma unroll
        for (int u = 0; u < 4; u++) {
            float f[VEC];
            V::widen(x[u], f);
#pragma unroll
            for (uint32_t i = 0; i < VEC; i++) a = __builtin_fmaf(f[i], f[i], a);
        }
        if (tid < head + tail) {
            const float f = V::widen1(ld_elem<E>(g, tid < head ? tid : head + nvec * VEC + (tid - head)));
            a = __builtin_fmaf(f, f, a);
        }
        sum += (double)a;
    }
    sum = wave_sum(sum);
    if ((tid & 63u) == 0) part[tid >> 6] = sum;
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

// The largest of a value over the 32 lanes that hold one block.
__device__ __forceinline__ float block_max(float x) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor(x, d, 64));
    return x;
}
__device__ __forceinline__ float finite_magnitude(float x) {
    const float a = fabsf(x);
    return a < __builtin_inff() ? a : 0.0f;
}
// the byte s for a block whose largest value is `largest`: TOP and MANT say that the format's largest value is
// 2^TOP * (1 + MANT / 2^23)
template <uint32_t TOP, uint32_t MANT>
__device__ __forceinline__ uint32_t state_scale(float largest) {
    const uint32_t b = as_u32(largest);
    const int s = (int)(b >> 23) - (int)TOP + ((b & 0x7fffffu) > MANT ? 1 : 0);
    return s < 1 ? 1u : (uint32_t)s;
}
__device__ __forceinline__ uint32_t scale_avg(float largest) { return state_scale<8, 0x600000>(largest); }       // 448
__device__ __forceinline__ uint32_t scale_sq(float largest) { return state_scale<18, 0x700000>(largest); }       // 30 * 2^14

// fp32 bits to a code of SHIFT bits less: nearest even, or up with the probability of what is cut off (16 random bits)
template <int SHIFT, bool RANDOM>
__device__ __forceinline__ uint32_t round_bits(uint32_t b, uint32_t random16) {
    if (RANDOM) return (b + (random16 << (SHIFT - 16))) >> SHIFT;
    return (b + ((1u << (SHIFT - 1)) - 1) + ((b >> SHIFT) & 1u)) >> SHIFT;
}
template <bool RANDOM>
__device__ __forceinline__ uint32_t code_avg(float m, uint32_t s, uint32_t random16) {
    const uint32_t c = round_bits<20, RANDOM>(as_u32(__builtin_ldexpf(fabsf(m), 7 - (int)s)), random16);
    return (fabsf(m) < __builtin_inff() ? c : 0x7fu) | ((as_u32(m) >> 24) & 0x80u);
}
template <bool RANDOM>
__device__ __forceinline__ uint32_t code_sq(float v, uint32_t s, uint32_t random16) {
    uint32_t c = round_bits<19, RANDOM>(as_u32(__builtin_ldexpf(fabsf(v), -3 - (int)s)), random16);
    if (c == 0 && v > 0.0f) c = 1;
    return v >= 0.0f && v < __builtin_inff() ? c : 255u;
}
__device__ __forceinline__ float value_avg(uint32_t code, uint32_t s) {
    const float f = __builtin_ldexpf(as_f32((code & 0x7fu) << 20), (int)s - 7);
    return as_f32(as_u32((code & 0x7fu) == 0x7fu ? __builtin_nanf("") : f) | ((code & 0x80u) << 24));
}
__device__ __forceinline__ float value_sq(uint32_t code, uint32_t s) {
    return code == 255u ? __builtin_nanf("") : __builtin_ldexpf(as_f32(code << 19), (int)s + 3);
}

// 32 random bits of an element: a multiply-and-shift mix of its index in the layout and the step's key.
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
__device__ __forceinline__ uint32_t element_random(uint64_t index, uint32_t key) {
    return mix32((uint32_t)index ^ key ^ ((uint32_t)(index >> 32) * 0x85EBCA77u));
}

// ---- a lane's eight elements ----------------------------------------------------------------------------------------------

template <class V>
__device__ __forceinline__ void load8(const void* p, uint32_t n, float* f) {
    typedef typename V::elem_t E;
    constexpr int VEC = V::VEC;
    if (n == kLaneElems) {
#pragma unroll
        for (int q = 0; q < (int)kLaneElems / VEC; q++) V::widen(ld_loose((const u32x4_u*)p + q), f + q * VEC);
    }
    else {
#pragma unroll
        for (uint32_t i = 0; i < kLaneElems; i++) f[i] = i < n ? V::widen1(ld_elem<E>(p, i)) : 0.0f;
    }
}
template <class V>
__device__ __forceinline__ void store8(void* p, uint32_t n, const float* f) {
    typedef typename V::elem_t E;
    constexpr int VEC = V::VEC;
    if (n == kLaneElems) {
#pragma unroll
        for (int q = 0; q < (int)kLaneElems / VEC; q++) st_loose((u32x4_u*)p + q, V::narrow(f + q * VEC));
    }
    else {
#pragma unroll
        for (uint32_t i = 0; i < kLaneElems; i++)
            if (i < n) st_elem<E>(p, i, V::narrow1(f[i]));
    }
}
// eight codes; a block starts on a multiple of 256 codes, so whole groups are aligned to the base's alignment
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_u __attribute__((aligned(1)));
__device__ __forceinline__ void load_codes(const uint8_t* p, uint32_t n, uint32_t* c) {
    if (n == kLaneElems) {
        const u32x2 x = __builtin_nontemporal_load((const u32x2_u*)p);
#pragma unroll
        for (int i = 0; i < 8; i++) c[i] = (x[i / 4] >> (8 * (i & 3))) & 0xffu;
    }
    else {
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) c[i] = i < n ? p[i] : 0;
    }
}
__device__ __forceinline__ void store_codes(uint8_t* p, uint32_t n, const uint32_t* c) {
    if (n == kLaneElems) {
        u32x2 x = { 0, 0 };
#pragma unroll
        for (int i = 0; i < 8; i++) x[i / 4] |= c[i] << (8 * (i & 3));
        __builtin_nontemporal_store(x, (u32x2_u*)p);
    }
    else {
#pragma unroll
        for (uint32_t i = 0; i < 8; i++)
            if (i < n) p[i] = (uint8_t)c[i];
    }
}

// ---- AdamW --------------------------------------------------------------------------------------------------------------

struct AdamwScalars {
    float beta1, rest1, beta2, rest2, eps;
    float decay;            // 1 - lr wd
    float step_size;        // lr / (1 - beta1^t)
    float root_scale;       // 1 / sqrt(1 - beta2^t)
    uint32_t key;           // of the step's random bits
    // on the device, where the host does not know them: the learning rate, the step, the factor of the gradients
    const float* lr_ptr;
    const int64_t* step_ptr;
    const float* grad_scale;
    double lr, weight_decay, beta1_d, beta2_d;
    int64_t step;
    uint64_t seed;
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
__host__ __device__ inline void adamw_derive(AdamwScalars& a) {
    a.decay = (float)(1.0 - a.lr * a.weight_decay);
    a.step_size = (float)(a.lr / (1.0 - whole_power(a.beta1_d, a.step)));
    a.root_scale = (float)(1.0 / sqrt(1.0 - whole_power(a.beta2_d, a.step)));
    a.key = step_key(a.seed, (uint64_t)a.step);
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

enum { STATE_FP32 = 0, STATE_NEAREST = 1, STATE_RANDOM = 2 };

// A block of threads takes 2048 elements of one item, a lane eight of them in a row.
template <class P, class G, bool MASTER, int STATE>
__global__ void __launch_bounds__(kBlock)
fusion_adamw_kernel(FusionPtrs params, FusionPtrs grads, const unsigned char* buffer, AdamwTables tb, AdamwState st, AdamwScalars a) {
    constexpr uint32_t GS = sizeof(typename G::elem_t), PS = sizeof(typename P::elem_t);
    constexpr uint32_t kItemElems = kFusionChunk / GS, kSubs = kItemElems / kOptTile;
    float scale = 1.0f;
    if (a.grad_scale) {
        scale = *a.grad_scale;
        if (!(fabsf(scale) < __builtin_inff())) return;         // gradients that are not finite: no step
    }
    if (a.lr_ptr || a.step_ptr) {
        if (a.lr_ptr) a.lr = (double)*a.lr_ptr;
        if (a.step_ptr) a.step = *a.step_ptr;
        adamw_derive(a);
    }
    const FusionItem w = tb.items[blockIdx.x / kSubs];
    const uint64_t e0 = (uint64_t)w.c * kItemElems + (blockIdx.x % kSubs) * kOptTile;
    const uint64_t count = tb.bytes[w.t] / GS;
    if (e0 >= count) return;
    const uint64_t e = e0 + threadIdx.x * kLaneElems;
    const uint32_t n = e >= count ? 0u : count - e < kLaneElems ? (uint32_t)(count - e) : kLaneElems;
    const uint64_t at = tb.off[w.t] / GS + e;                   // the lane's first element in the plan's layout
    unsigned char* p = (unsigned char*)(uintptr_t)params.get(w.t - tb.t0) + e * PS;
    const unsigned char* gp = (buffer ? buffer + tb.off[w.t] : (const unsigned char*)(uintptr_t)grads.get(w.t - tb.t0)) + e * GS;

    float g[8], m[8], v[8], x[8];
    load8<G>(gp, n, g);
    if (MASTER) load8<F32Vec>(st.master + at, n, x);
    else load8<P>(p, n, x);
    if (STATE == STATE_FP32) {
        load8<F32Vec>((const float*)st.avg + at, n, m);
        load8<F32Vec>((const float*)st.sq + at, n, v);
    }
    else {
        uint32_t cm[8], cv[8], sm = 0, sv = 0;
        load_codes((const uint8_t*)st.avg + at, n, cm);
        load_codes((const uint8_t*)st.sq + at, n, cv);
        if (n) {
            const uint8_t* s = st.scales + 2 * (at / kStateBlock);
            sm = s[0];
            sv = s[1];
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            m[i] = value_avg(cm[i], sm);
            v[i] = value_sq(cv[i], sv);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float gs = g[i] * scale;
        m[i] = m[i] * a.beta1 + gs * a.rest1;
        v[i] = v[i] * a.beta2 + (gs * gs) * a.rest2;
        const float root = sqrtf(v[i]) * a.root_scale + a.eps;
        x[i] = x[i] * a.decay - (m[i] / root) * a.step_size;
    }
    if (MASTER) store8<F32Vec>(st.master + at, n, x);
    store8<P>(p, n, x);
    if (STATE == STATE_FP32) {
        store8<F32Vec>((float*)st.avg + at, n, m);
        store8<F32Vec>((float*)st.sq + at, n, v);
    }
    else {
        float lm = 0.0f, lv = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            if (i < n) {
                lm = fmaxf(lm, finite_magnitude(m[i]));
                lv = fmaxf(lv, finite_magnitude(v[i]));
            }
        }
        const uint32_t sm = scale_avg(block_max(lm)), sv = scale_sq(block_max(lv));
        uint32_t cm[8], cv[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t r = STATE == STATE_RANDOM ? element_random(at + i, a.key) : 0;
            cm[i] = code_avg<STATE == STATE_RANDOM>(m[i], sm, r & 0xffffu);
            cv[i] = code_sq<STATE == STATE_RANDOM>(v[i], sv, r >> 16);
        }
        store_codes((uint8_t*)st.avg + at, n, cm);
        store_codes((uint8_t*)st.sq + at, n, cv);
        if (n && (threadIdx.x & 31u) == 0) {
            uint8_t* s = st.scales + 2 * (at / kStateBlock);
            s[0] = (uint8_t)sm;
            s[1] = (uint8_t)sv;
        }
    }
}

// ---- 8-bit states in and out ----------------------------------------------------------------------------------------------

// The values of the codes, as fp32 or bfloat16 (which holds every one of them from 2^-126 up).
template <class V>
__global__ void __launch_bounds__(kBlock)
state_decode_kernel(AdamwTables tb, uint32_t item_elems, const uint8_t* avg, const uint8_t* sq, const uint8_t* scales,
                    typename V::elem_t* out_avg, typename V::elem_t* out_sq) {
    const uint32_t subs = item_elems / kOptTile;
    const FusionItem w = tb.items[blockIdx.x / subs];
    const uint64_t e = (uint64_t)w.c * item_elems + (blockIdx.x % subs) * kOptTile + threadIdx.x * kLaneElems;
    const uint64_t count = tb.bytes[w.t] >> tb.log_esize;
    if (e >= count) return;
    const uint32_t n = count - e < kLaneElems ? (uint32_t)(count - e) : kLaneElems;
    const uint64_t at = (tb.off[w.t] >> tb.log_esize) + e;
    uint32_t cm[8], cv[8];
    float m[8], v[8];
    load_codes(avg + at, n, cm);
    load_codes(sq + at, n, cv);
    const uint32_t sm = scales[2 * (at / kStateBlock)], sv = scales[2 * (at / kStateBlock) + 1];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        m[i] = value_avg(cm[i], sm);
        v[i] = value_sq(cv[i], sv);
    }
    store8<V>(out_avg + at, n, m);
    store8<V>(out_sq + at, n, v);
}

// fp32 or bfloat16 values to codes, rounded to nearest.
template <class V>
__global__ void __launch_bounds__(kBlock)
state_encode_kernel(AdamwTables tb, uint32_t item_elems, const typename V::elem_t* in_avg, const typename V::elem_t* in_sq, uint8_t* avg,
                    uint8_t* sq, uint8_t* scales) {
    const uint32_t subs = item_elems / kOptTile;
    const FusionItem w = tb.items[blockIdx.x / subs];
    const uint64_t e = (uint64_t)w.c * item_elems + (blockIdx.x % subs) * kOptTile + threadIdx.x * kLaneElems;
    const uint64_t count = tb.bytes[w.t] >> tb.log_esize;
    const uint32_t n = e >= count ? 0u : count - e < kLaneElems ? (uint32_t)(count - e) : kLaneElems;
    const uint64_t at = (tb.off[w.t] >> tb.log_esize) + e;
    float m[8], v[8], lm = 0.0f, lv = 0.0f;
    load8<V>(in_avg + at, n, m);
    load8<V>(in_sq + at, n, v);
#pragma unroll
    for (uint32_t i = 0; i < 8; i++) {
        lm = fmaxf(lm, finite_magnitude(m[i]));
        lv = fmaxf(lv, finite_magnitude(v[i]));
    }
    const uint32_t sm = scale_avg(block_max(lm)), sv = scale_sq(block_max(lv));
    uint32_t cm[8], cv[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        cm[i] = code_avg<false>(m[i], sm, 0);
        cv[i] = code_sq<false>(v[i], sv, 0);
    }
    store_codes(avg + at, n, cm);
    store_codes(sq + at, n, cv);
    if (n && (threadIdx.x & 31u) == 0) {
        scales[2 * (at / kStateBlock)] = (uint8_t)sm;
        scales[2 * (at / kStateBlock) + 1] = (uint8_t)sv;
    }
}

}  // namespace mi
