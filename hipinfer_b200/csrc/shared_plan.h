// What the planner of the shared-prefix attention hands to its kernels (shared_plan.cu, attention_shared*.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

// Keys [lo, hi) of one kv head against `tokens` consecutive rows of q with all heads of the group: read through block table row
// `table`. `pos` is the position of the first token where a row sees no key behind its own position, SP_NO_MASK where all rows see
// all keys of the range. Row i * G + g of the item is part row part + i * G + g of the workspace.
struct SharedItem {
  int table, token, tokens, pos, lo, hi, head, part;
};
// What a row of q is put together from: parts [k] of the shared range and of its request's own, the (kv head h, head g of its group)
// row being base + (h * n + k) * rows + g, and the keys of this step's own rows, positions first .. first + fresh - 1.
struct SharedToken {
  int pre_base, pre_n, pre_rows, own_base, own_n, own_rows, table, first, fresh, pad[3];
};
constexpr int SP_HEADER = 16;
enum { SP_ITEMS, SP_CTAS, SP_PARTS, SP_TOKENS, SP_MAX_ROWS, SP_OFF_ITEMS, SP_OFF_CTAS, SP_OFF_TOKENS, SP_INTS, SP_MASKED };
constexpr int SP_NO_MASK = 1 << 30;
// A request of up to this many rows in the step has its rows' own keys (they are causal among themselves) added by the joining kernel; the
// items then have no mask, and what stands behind a row, whatever it is, is never multiplied by a probability of 0.
constexpr int SP_FRESH = 16;

// The items on the tensor cores (attention_shared_tc.cu): bfloat16, for a plan whose items have up to 2 * (128 / G) tokens, of which those of up to
// 128 / G leave two parts. masked: whether any of them has a `pos`. scale_log2: the scale times log2(e).
int hb_shared_items_tc(const void* q, long ldq, const void* kc, const void* vc, long num_pages, const int* bt, int bt_stride, const SharedItem* items,
                       const int* cta_items, int ctas, int masked, int T, float* part_o, float2* part_ml, int Hq, int Hkv, int D, int page_size, float scale_log2, int* status, cudaStream_t s);
