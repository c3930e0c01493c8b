// Entry points of the optimizer operators on a fusion plan (gradient norm, AdamW step, 8-bit states) in libmi_ccl_comp.so.
#include <hip/hip_runtime.h>

#include "../../include/mi_ccl_comp.h"
#include "fusion_plan.hpp"
#include "launch_geometry.hpp"
#include "optimizer_kernels.hpp"

using namespace mi;

namespace {

bool float_type(int dtype) {
    return dtype == MI_CCL_FLOAT32 || dtype == MI_CCL_FLOAT16 || dtype == MI_CCL_BFLOAT16;
}

// A device address that the kernels' 48-bit tables hold, at a multiple of the element size.
bool address_ok(const void* p, size_t esz) {
    return p && (uintptr_t)p % esz == 0 && ((uint64_t)(uintptr_t)p >> 48) == 0;
}

// the gradients of a call: every tensor of its own, or one fusion buffer in the plan's layout
bool gradients_ok(const mi_ccl_fusion_plan* plan, const void* const* grads, const void* fusion_buf) {
    if ((grads != nullptr) == (fusion_buf != nullptr))
        return plan->total_bytes == 0;
    if (fusion_buf)
        return (uintptr_t)fusion_buf % plan->esz == 0;
    for (size_t t = 0; t < plan->k; t++)
        if (plan->counts[t] && !address_ok(grads[t], plan->esz))
            return false;
    return true;
}

void set_pointers(FusionPtrs& to, const void* const* from, size_t t0, size_t t1) {
    for (size_t t = t0; t < t1; t++) to.set(t - t0, from[t]);      // the address of an empty tensor may be anything: it is not used
}

// ---- norm

// blocks of the launch over tensors [t0, t1)
uint32_t norm_blocks(const mi_ccl_fusion_plan* plan, size_t t0, size_t t1) {
    const uint64_t items = plan->item_begin[t1] - plan->item_begin[t0];
    return (uint32_t)(items < kNormBlocks ? items : kNormBlocks);
}
size_t norm_groups(const mi_ccl_fusion_plan* plan) {
    return (plan->k + kFusionGroup - 1) / kFusionGroup;
}

template <class V>
hipError_t norm_launch(bool buffer_form, uint32_t blocks, hipStream_t stream, const FusionPtrs& ptrs, const void* buffer, const NormTables& tb, double* partial) {
    if (buffer_form)
        hipLaunchKernelGGL((fusion_norm_kernel<V, true>), dim3(blocks), dim3(kBlock), 0, stream, ptrs, (const unsigned char*)buffer, tb, partial);
    else
        hipLaunchKernelGGL((fusion_norm_kernel<V, false>), dim3(blocks), dim3(kBlock), 0, stream, ptrs, (const unsigned char*)nullptr, tb, partial);
    return hipGetLastError();
}
hipError_t norm_by_type(int dtype, bool buffer_form, uint32_t blocks, hipStream_t stream, const FusionPtrs& ptrs, const void* buffer,
                        const NormTables& tb, double* partial) {
    if (dtype == MI_CCL_FLOAT32) return norm_launch<F32Vec>(buffer_form, blocks, stream, ptrs, buffer, tb, partial);
    if (dtype == MI_CCL_BFLOAT16) return norm_launch<Bf16Vec>(buffer_form, blocks, stream, ptrs, buffer, tb, partial);
    return norm_launch<Fp16Vec>(buffer_form, blocks, stream, ptrs, buffer, tb, partial);
}

// ---- AdamW

struct AdamwLaunch {
    uint32_t blocks;
    hipStream_t stream;
    const FusionPtrs *params, *grads;
    const unsigned char* buffer;
    AdamwTables tb;
    AdamwState st;
    AdamwScalars sc;
};
template <class P, class G, bool MASTER, int STATE>
hipError_t adamw_launch(const AdamwLaunch& a) {
    hipLaunchKernelGGL((fusion_adamw_kernel<P, G, MASTER, STATE>), dim3(a.blocks), dim3(kAdamwBlock), 0, a.stream, *a.params, *a.grads, a.buffer, a.tb,
                       a.st, a.sc);
    return hipGetLastError();
}
template <class P, class G, bool MASTER>
hipError_t adamw_by_state(int state, const AdamwLaunch& a) {
    if (state == STATE_FP32) return adamw_launch<P, G, MASTER, STATE_FP32>(a);
    if (state == STATE_NEAREST) return adamw_launch<P, G, MASTER, STATE_NEAREST>(a);
    return adamw_launch<P, G, MASTER, STATE_RANDOM>(a);
}
template <class P, bool MASTER>
hipError_t adamw_by_grad(int dtype, int state, const AdamwLaunch& a) {
    if (dtype == MI_CCL_FLOAT32) return adamw_by_state<P, F32Vec, MASTER>(state, a);
    if (dtype == MI_CCL_BFLOAT16) return adamw_by_state<P, Bf16Vec, MASTER>(state, a);
    return adamw_by_state<P, Fp16Vec, MASTER>(state, a);
}
hipError_t adamw_by_type(int param_dtype, bool master, int dtype, int state, const AdamwLaunch& a) {
    if (param_dtype == MI_CCL_FLOAT32) return adamw_by_grad<F32Vec, false>(dtype, state, a);
    if (param_dtype == MI_CCL_BFLOAT16)
        return master ? adamw_by_grad<Bf16Vec, true>(dtype, state, a) : adamw_by_grad<Bf16Vec, false>(dtype, state, a);
    return master ? adamw_by_grad<Fp16Vec, true>(dtype, state, a) : adamw_by_grad<Fp16Vec, false>(dtype, state, a);
}

// every tensor starts on a block of 256 elements: what the 8-bit states need of the layout
bool blocks_aligned(const mi_ccl_fusion_plan* plan) {
    for (size_t t = 0; t < plan->k; t++)
        if (plan->offsets[t] % (plan->esz * kStateBlock)) return false;
    return true;
}

AdamwTables plan_tables(const mi_ccl_fusion_plan* plan) {
    AdamwTables tb;
    tb.off = plan->d_off;
    tb.bytes = plan->d_bytes;
    tb.items = plan->d_items;
    tb.t0 = 0;
    tb.log_esize = plan->esz == 4 ? 2 : 1;
    return tb;
}

// the most items of one launch whose blocks take `subs` parts of an item each
uint64_t items_per_launch(uint32_t subs) {
    return hip_block_limit(kBlock) / subs;
}

int state_check(const mi_ccl_fusion_plan* plan, int value_dtype, const void* avg, const void* sq, const void* scales, const void* value_avg,
                const void* value_sq) {
    if (!plan || !float_type(plan->dtype) || (value_dtype != MI_CCL_FLOAT32 && value_dtype != MI_CCL_BFLOAT16) || !blocks_aligned(plan))
        return MI_CCL_INVALID_ARGUMENTS;
    if (plan->total_bytes && (!avg || !sq || !scales || !value_avg || !value_sq ||
                              ((uintptr_t)value_avg | (uintptr_t)value_sq) % fusion_dtype_size(value_dtype)))
        return MI_CCL_INVALID_ARGUMENTS;
    return MI_CCL_SUCCESS;
}

}  // namespace

extern "C" {

size_t mi_ccl_fusion_plan_elements(const mi_ccl_fusion_plan* plan) {
    return plan ? plan->total_bytes / plan->esz : 0;
}

size_t mi_ccl_fusion_norm_workspace(const mi_ccl_fusion_plan* plan) {
    if (!plan)
        return 0;
    const uint64_t items = plan->item_begin[plan->k];
    const uint64_t most = (uint64_t)norm_groups(plan) * kNormBlocks;
    return (size_t)(items < most ? items : most) * sizeof(double);
}

int mi_ccl_fusion_norm(mi_ccl_fusion_plan* plan, const void* const* grads, const void* fusion_buf, double multiplier, double max_norm,
                       float* result, void* workspace, size_t workspace_bytes, void* stream) {
    if (!plan || !float_type(plan->dtype) || !result || (uintptr_t)result % sizeof(float) || multiplier != multiplier || max_norm != max_norm ||
        !gradients_ok(plan, grads, fusion_buf))
        return MI_CCL_INVALID_ARGUMENTS;
    const size_t need = mi_ccl_fusion_norm_workspace(plan);
    if (need && (!workspace || (uintptr_t)workspace % sizeof(double) || workspace_bytes < need))
        return MI_CCL_INVALID_ARGUMENTS;
    double* partial = (double*)workspace;
    uint32_t n = 0;
    FusionPtrs ptrs = {};
    // a fusion buffer needs no table of pointers: all its tensors are one launch
    const size_t group = fusion_buf ? plan->k : (size_t)kFusionGroup;
    for (size_t t0 = 0; t0 < plan->k; t0 += group) {
        const size_t t1 = (t0 + group < plan->k) ? t0 + group : plan->k;
        const uint32_t blocks = norm_blocks(plan, t0, t1);
        if (blocks == 0)
            continue;
        if (!fusion_buf)
            set_pointers(ptrs, grads, t0, t1);
        NormTables tb = { plan->d_off, plan->d_bytes, plan->d_items + plan->item_begin[t0],
                          (uint32_t)(plan->item_begin[t1] - plan->item_begin[t0]), (uint32_t)t0 };
        g_last_kernel = "fusion_norm_kernel";
        const hipError_t e = norm_by_type(plan->dtype, fusion_buf != nullptr, blocks, (hipStream_t)stream, ptrs, fusion_buf, tb, partial + n);
        if (e != hipSuccess)
            return fusion_status_of(e);
        n += blocks;
    }
    hipLaunchKernelGGL(fusion_norm_finish_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, (const double*)partial, n, multiplier, max_norm,
                       result);
    return fusion_status_of(hipGetLastError());
}

int mi_ccl_fusion_adamw(mi_ccl_fusion_plan* plan, int param_dtype, void* const* params, const void* const* grads, const void* fusion_buf,
                        int state_format, void* exp_avg, void* exp_avg_sq, void* scales, float* master, const mi_ccl_adamw_options* o,
                        void* stream) {
    if (!plan || !float_type(plan->dtype) || !float_type(param_dtype) || !params || !o || !gradients_ok(plan, grads, fusion_buf))
        return MI_CCL_INVALID_ARGUMENTS;
    const bool eight = state_format == MI_CCL_STATE_8BIT;
    if (!eight && state_format != MI_CCL_STATE_FP32)
        return MI_CCL_INVALID_ARGUMENTS;
    // what makes no sense is refused; the comparisons are false for NaN
    if (!(o->lr >= 0.0) || !(o->beta1 >= 0.0 && o->beta1 < 1.0) || !(o->beta2 >= 0.0 && o->beta2 < 1.0) || !(o->eps >= 0x1p-126) ||
        !(o->weight_decay >= 0.0) || (!o->step_ptr && o->step < 1) || (o->stochastic != 0 && (o->stochastic != 1 || !eight)))
        return MI_CCL_INVALID_ARGUMENTS;
    if ((uintptr_t)o->step_ptr % sizeof(int64_t) || (uintptr_t)o->lr_ptr % sizeof(float) || (uintptr_t)o->grad_scale % sizeof(float))
        return MI_CCL_INVALID_ARGUMENTS;
    if ((o->step_ptr || o->lr_ptr) && (!o->workspace || (uintptr_t)o->workspace % alignof(AdamwDerived)))
        return MI_CCL_INVALID_ARGUMENTS;
    if (master && param_dtype == MI_CCL_FLOAT32)
        return MI_CCL_INVALID_ARGUMENTS;
    if (eight && (!blocks_aligned(plan) || (plan->total_bytes && !scales)))
        return MI_CCL_INVALID_ARGUMENTS;
    if (plan->total_bytes && (!exp_avg || !exp_avg_sq))
        return MI_CCL_INVALID_ARGUMENTS;
    if ((!eight && ((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) % sizeof(float)) || (uintptr_t)master % sizeof(float))
        return MI_CCL_INVALID_ARGUMENTS;
    const size_t psize = fusion_dtype_size(param_dtype);
    for (size_t t = 0; t < plan->k; t++)
        if (plan->counts[t] && !address_ok(params[t], psize))
            return MI_CCL_INVALID_ARGUMENTS;

    FusionPtrs pp = {}, gg = {};
    AdamwLaunch a;
    a.stream = (hipStream_t)stream;
    a.params = &pp;
    a.grads = &gg;
    a.buffer = (const unsigned char*)fusion_buf;
    a.tb = plan_tables(plan);
    a.st = AdamwState{ exp_avg, exp_avg_sq, (uint8_t*)scales, master };
    AdamwScalars& sc = a.sc;
    sc.beta1 = (float)o->beta1;
    sc.rest1 = (float)(1.0 - o->beta1);
    sc.beta2 = (float)o->beta2;
    sc.rest2 = (float)(1.0 - o->beta2);
    sc.eps = (float)o->eps;
    sc.grad_scale = o->grad_scale;
    const AdamwHyper h = { o->lr, o->weight_decay, o->beta1, o->beta2, o->step_ptr ? 1 : o->step, o->seed };
    sc.d = adamw_derive(h);
    sc.derived = nullptr;
    if ((o->step_ptr || o->lr_ptr) && plan->item_begin[plan->k]) {
        AdamwDerived* derived = (AdamwDerived*)o->workspace;
        g_last_kernel = "adamw_derive_kernel";
        hipLaunchKernelGGL(adamw_derive_kernel, dim3(1), dim3(1), 0, (hipStream_t)stream, h, o->lr_ptr, o->step_ptr, derived);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess)
            return fusion_status_of(e);
        sc.derived = derived;
    }

    const int state = !eight ? STATE_FP32 : o->stochastic ? STATE_RANDOM : STATE_NEAREST;
    const uint32_t subs = kFusionChunk / (uint32_t)plan->esz / kAdamwTile;
    const uint64_t most = items_per_launch(subs);
    for (size_t t0 = 0; t0 < plan->k; t0 += kFusionGroup) {
        const size_t t1 = (t0 + kFusionGroup < plan->k) ? t0 + kFusionGroup : plan->k;
        set_pointers(pp, (const void* const*)params, t0, t1);
        if (!fusion_buf && grads)
            set_pointers(gg, grads, t0, t1);
        a.tb.t0 = (uint32_t)t0;
        for (uint64_t i0 = plan->item_begin[t0]; i0 < plan->item_begin[t1]; i0 += most) {
            const uint64_t i1 = (i0 + most < plan->item_begin[t1]) ? i0 + most : plan->item_begin[t1];
            a.tb.items = plan->d_items + i0;
            a.blocks = (uint32_t)((i1 - i0) * subs);
            g_last_kernel = "fusion_adamw_kernel";
            const hipError_t e = adamw_by_type(param_dtype, master != nullptr, plan->dtype, state, a);
            if (e != hipSuccess)
                return fusion_status_of(e);
        }
    }
    return MI_CCL_SUCCESS;
}

int mi_ccl_fusion_state_decode(mi_ccl_fusion_plan* plan, const void* exp_avg, const void* exp_avg_sq, const void* scales, int value_dtype,
                               void* values_avg, void* values_sq, void* stream) {
    const int rc = state_check(plan, value_dtype, exp_avg, exp_avg_sq, scales, values_avg, values_sq);
    if (rc != MI_CCL_SUCCESS)
        return rc;
    AdamwTables tb = plan_tables(plan);
    const uint32_t elems = kFusionChunk / (uint32_t)plan->esz, subs = elems / (kBlock * 4 * kDecodeGroups);
    const uint64_t most = items_per_launch(subs), all = plan->item_begin[plan->k];
    for (uint64_t i0 = 0; i0 < all; i0 += most) {
        tb.items = plan->d_items + i0;
        const dim3 grid((unsigned)((i0 + most < all ? most : all - i0) * subs));
        g_last_kernel = "state_decode_kernel";
        if (value_dtype == MI_CCL_FLOAT32)
            hipLaunchKernelGGL((state_decode_kernel<F32Vec>), grid, dim3(kBlock), 0, (hipStream_t)stream, tb, elems, (const uint8_t*)exp_avg,
                               (const uint8_t*)exp_avg_sq, (const uint8_t*)scales, (uint32_t*)values_avg, (uint32_t*)values_sq);
        else
            hipLaunchKernelGGL((state_decode_kernel<Bf16Vec>), grid, dim3(kBlock), 0, (hipStream_t)stream, tb, elems, (const uint8_t*)exp_avg,
                               (const uint8_t*)exp_avg_sq, (const uint8_t*)scales, (uint16_t*)values_avg, (uint16_t*)values_sq);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess)
            return fusion_status_of(e);
    }
    return MI_CCL_SUCCESS;
}

int mi_ccl_fusion_state_encode(mi_ccl_fusion_plan* plan, int value_dtype, const void* values_avg, const void* values_sq, void* exp_avg,
                               void* exp_avg_sq, void* scales, void* stream) {
    const int rc = state_check(plan, value_dtype, exp_avg, exp_avg_sq, scales, values_avg, values_sq);
    if (rc != MI_CCL_SUCCESS)
        return rc;
    AdamwTables tb = plan_tables(plan);
    const uint32_t elems = kFusionChunk / (uint32_t)plan->esz, subs = elems / (kBlock * 4 * kEncodeGroups);
    const uint64_t most = items_per_launch(subs), all = plan->item_begin[plan->k];
    for (uint64_t i0 = 0; i0 < all; i0 += most) {
        tb.items = plan->d_items + i0;
        const dim3 grid((unsigned)((i0 + most < all ? most : all - i0) * subs));
        g_last_kernel = "state_encode_kernel";
        if (value_dtype == MI_CCL_FLOAT32)
            hipLaunchKernelGGL((state_encode_kernel<F32Vec>), grid, dim3(kBlock), 0, (hipStream_t)stream, tb, elems, (const uint32_t*)values_avg,
                               (const uint32_t*)values_sq, (uint8_t*)exp_avg, (uint8_t*)exp_avg_sq, (uint8_t*)scales);
        else
            hipLaunchKernelGGL((state_encode_kernel<Bf16Vec>), grid, dim3(kBlock), 0, (hipStream_t)stream, tb, elems, (const uint16_t*)values_avg,
                               (const uint16_t*)values_sq, (uint8_t*)exp_avg, (uint8_t*)exp_avg_sq, (uint8_t*)scales);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess)
            return fusion_status_of(e);
    }
    return MI_CCL_SUCCESS;
}

} /* extern "C" */
