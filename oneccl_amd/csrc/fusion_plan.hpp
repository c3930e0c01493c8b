// A fused group's layout and its device-side work table: what mi_ccl_fusion_plan_create makes and the entry points of
// fusion.hip (pack, unpack, fused reduce) and optimizer.hip (norm, AdamW step, 8-bit states) read.
#pragma once

#include <vector>

#include "../../include/mi_ccl_comp.h"
#include "fusion_kernels.hpp"

namespace mi {

inline int fusion_status_of(hipError_t e) {
    if (e == hipSuccess)
        return MI_CCL_SUCCESS;
    if (e == hipErrorOutOfMemory)
        return MI_CCL_OUT_OF_RESOURCE;
    if (e == hipErrorInvalidValue)
        return MI_CCL_INVALID_ARGUMENTS;
    return MI_CCL_RUNTIME_ERROR;
}

inline size_t fusion_dtype_size(int dtype) {
    static const size_t sz[MI_CCL_DATATYPE_LAST] = { 1, 1, 2, 2, 4, 4, 8, 8, 2, 4, 8, 2 };
    return (dtype >= 0 && dtype < MI_CCL_DATATYPE_LAST) ? sz[dtype] : 0;
}

}  // namespace mi

struct mi_ccl_fusion_plan {
    size_t k = 0;
    int dtype = 0;
    size_t esz = 0;
    size_t align = 1;
    size_t total_bytes = 0;
    std::vector<size_t> counts;
    std::vector<size_t> offsets;           // bytes
    std::vector<uint64_t> item_begin;      // k + 1
    std::vector<uint64_t> tile_begin;      // k + 1: tiles of kFusionTile bytes
    void* d_table = nullptr;               // [off: k x u64][bytes: k x u64][items][tile_end: k x u32]
    const uint64_t* d_off = nullptr;
    const uint64_t* d_bytes = nullptr;
    const mi::FusionItem* d_items = nullptr;
    const uint32_t* d_tile_end = nullptr;
};
