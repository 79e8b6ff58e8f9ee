// The cache operators' host side: checked arguments turned into kernel views, and the launches. The C
// entry points (cache_ops.hip) and the batched runtime call these.
#pragma once

#include "cache_device.hpp"
#include "host_common.hpp"

namespace stamd {

CacheView cache_view(const st_kv_cache* cache);
RowsView rows_view(const st_kv_cache* cache, const st_new_rows* rows);
void append_rows(const st_kv_cache* cache, const st_new_rows* rows, const st_append_args* args, hipStream_t stream);
// Bytes that attend needs as its workspace.
size_t attention_workspace(const st_kv_cache* cache, const st_new_rows* rows, int q_heads, int dtype);
// out_layout 1, 2: the output goes to a batch's operand layout of out_ld columns (act_index of FP32 and
// bfloat16 weights), rows being streams; FP32 only.
void attend_rows(const st_kv_cache* cache, const st_new_rows* rows, const st_attention_args* args, hipStream_t stream,
                 int out_layout = 0, int out_ld = 0);

}  // namespace stamd
