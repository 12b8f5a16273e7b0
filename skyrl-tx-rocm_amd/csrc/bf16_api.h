// Entry points of the torch layers' operators beside the quantized path: products grouped by expert in bf16, embedding rows and
// their gradient, the norm and the clipping of adapter gradients.  Conventions, status codes and streams are those of the public C
// header; like the group-scaled backward they are no part of it: another framework's binding brings its own operators here.
#pragma once
#include "../../include/mi355_w8a8.h"

extern "C" {

/*
 * Products grouped by expert with ragged sizes on bf16 weights (the ragged_dot of skyrl/tx/layers/util.py:8-59 that
 * LoRAExpert.__call__, skyrl/tx/layers/lora.py:394-444, makes of its unquantized kernels), and their two gradients:
 *   out[i]  = bf16(x[i] @ weight[g(i)])            dx[i] = bf16(dy[i] @ weight[g(i)]^T)
 *   dw[g]   = sum over the rows of g of x[i]^T dy[i]
 * with float32 sums.  Rows are sorted by group: group g owns group_sizes[g] rows behind those of the groups before it.
 * Rows behind the last group give zeros and take part in no sum; a group without rows has a zero dw.  Sizes are read
 * on the device and clamped to what the m rows hold.  k and n are multiples of 8, at most
 * MI355_W8A8_BF16_GROUPED_MAX_FEATURES; m at most 2^20, n_groups at most 1024.
 */
#define MI355_W8A8_BF16_GROUPED_MAX_FEATURES 65536u
/* tiles of the products (at most one of the three; default: by the rows, the groups and how many tiles result) */
#define MI355_W8A8_FLAG_BF16_GROUPED_TILE_256X256 4u
#define MI355_W8A8_FLAG_BF16_GROUPED_TILE_128X256 8u
#define MI355_W8A8_FLAG_BF16_GROUPED_TILE_64X128 16u
typedef struct mi355_w8a8_bf16_grouped_problem {
  uint32_t struct_size;     /* sizeof(mi355_w8a8_bf16_grouped_problem) */
  uint32_t flags;
  uint32_t m;               /* rows of x */
  uint32_t k;               /* in features */
  uint32_t n;               /* out features */
  uint32_t n_groups;
  const void* x;            /* bf16 [m, k] */
  const void* weight;       /* bf16 [n_groups, k, n] */
  const int32_t* group_sizes; /* int32 [n_groups] */
  void* out;                /* bf16 [m, n] */
  void* workspace;          /* 256-byte aligned device scratch; may be NULL where no bytes are needed */
  uint64_t workspace_bytes; /* >= mi355_w8a8_bf16_grouped_workspace_bytes(...) */
} mi355_w8a8_bf16_grouped_problem;
#define MI355_W8A8_FLAG_BF16_GROUPED_DW_F32 1u /* dw is float32 */
typedef struct mi355_w8a8_bf16_grouped_bwd_problem {
  uint32_t struct_size;     /* sizeof(mi355_w8a8_bf16_grouped_bwd_problem) */
  uint32_t flags;
  uint32_t m, k, n, n_groups; /* of the forward */
  const void* x;            /* bf16 [m, k]; for dw */
  const void* dy;           /* bf16 [m, n] */
  const void* weight;       /* bf16 [n_groups, k, n]; for dx */
  const int32_t* group_sizes; /* int32 [n_groups] */
  void* dx;                 /* bf16 [m, k], or NULL: not wanted */
  void* dw;                 /* bf16 or float32 [n_groups, k, n], or NULL: not wanted */
  void* workspace;          /* as above, for what dx and dw need one after the other */
  uint64_t workspace_bytes; /* >= mi355_w8a8_bf16_grouped_bwd_workspace_bytes(...) */
} mi355_w8a8_bf16_grouped_bwd_problem;
/* Scratch of a call: nothing, or the parts of a long contraction that few tiles share.  0 also for sizes that a call refuses. */
uint64_t mi355_w8a8_bf16_grouped_workspace_bytes(uint32_t m, uint32_t k, uint32_t n, uint32_t n_groups, uint32_t flags);
uint64_t mi355_w8a8_bf16_grouped_bwd_workspace_bytes(uint32_t m, uint32_t k, uint32_t n, uint32_t n_groups, uint32_t flags, uint32_t want_dx,
                                                     uint32_t want_dw);
/* The tiles (a flag) of a backward call that computes both gradients in one launch, 0: each has its own. */
uint32_t mi355_w8a8_bf16_grouped_bwd_joint_tile(uint32_t m, uint32_t k, uint32_t n, uint32_t n_groups, uint32_t flags);
int mi355_w8a8_bf16_grouped_v1(const mi355_w8a8_bf16_grouped_problem* problem, void* stream);
int mi355_w8a8_bf16_grouped_bwd_v1(const mi355_w8a8_bf16_grouped_bwd_problem* problem, void* stream);

/*
 * Rows of an embedding table, scaled, and the table's gradient by sorted tokens:
 *   mi355_w8a8_embedding_v1      out[t] = scale(t) * table[adapter(t)][ids[t]]
 *   mi355_w8a8_embedding_bwd_v1  out[a][v] = scale(a) * sum over t with adapter(t) = a, ids[t] = v of d_out[t], every
 *                                row of the table written, zeros where no token names it
 * in float32, rounded once, the sums in the order of the tokens (the same bits at every call).  With n_adapters = 0 the table
 * is [vocab, width] and `scale` counts; else it is [n_adapters, vocab, width], the A factors of a LoRA embedding, and scales
 * names one factor for each adapter (NULL: `scale` for all).  Tokens whose id or adapter is out of range read zeros and leave no
 * gradient.  n_tokens at most 2^20, width at most MI355_W8A8_EMBEDDING_MAX_WIDTH, rows of the table at most
 * MI355_W8A8_EMBEDDING_MAX_ROWS.
 */
#define MI355_W8A8_FLAG_EMBEDDING_F32 1u   /* table, out and d_out are float32, else bf16 */
#define MI355_W8A8_FLAG_EMBEDDING_IDS64 2u /* ids are int64, else int32 */
#define MI355_W8A8_EMBEDDING_MAX_WIDTH 65536u
#define MI355_W8A8_EMBEDDING_MAX_ROWS 0x40000000u
typedef struct mi355_w8a8_embedding_problem {
  uint32_t struct_size;     /* sizeof(mi355_w8a8_embedding_problem) */
  uint32_t flags;
  uint32_t n_tokens, vocab, width, n_adapters;
  float scale;
  uint32_t reserved;
  const void* table;        /* forward: the table */
  const void* d_out;        /* backward: [n_tokens, width] */
  const void* ids;          /* int32 or int64 [n_tokens] */
  const int32_t* adapter_indices; /* int32 [n_tokens], or NULL with at most one adapter */
  const float* scales;      /* f32 [n_adapters] or NULL */
  void* out;                /* forward: [n_tokens, width]; backward: the table's gradient, 16-byte aligned */
  void* workspace;          /* backward: 256-byte aligned device scratch */
  uint64_t workspace_bytes; /* >= mi355_w8a8_embedding_bwd_workspace_bytes(...) */
} mi355_w8a8_embedding_problem;
int mi355_w8a8_embedding_v1(const mi355_w8a8_embedding_problem* problem, void* stream);
uint64_t mi355_w8a8_embedding_bwd_workspace_bytes(uint32_t n_tokens, uint32_t vocab, uint32_t width, uint32_t n_adapters, uint32_t flags);
int mi355_w8a8_embedding_bwd_v1(const mi355_w8a8_embedding_problem* problem, void* stream);

/*
 * The global norm over many gradient tensors, one for each adapter (their leading axis; 1 for gradients of one model), and
 * clipping:
 *   norms[a] = sqrt(sum over the tensors of sum(grad[a]^2))        (double sums, the same bits at every call)
 *   out[a]   = grad[a] * (norms[a] > limits[a] ? limits[a] / norms[a] : 1)
 * A tensor's out may be its grad itself, other overlaps of the two are refused; different tensors must not overlap where one is written.  Where a norm or a limit is NaN that adapter's gradients stay as they are, a
 * negative limit counts as zero.  The tensor table is host memory and is read before the call returns; limits and norms are device
 * memory.  More than 16 tensors are found by the kernels in a table that the call writes into the workspace;
 * MI355_W8A8_FLAG_GRAD_TABLE_KEPT says that it is still there from an earlier call on the same workspace with the same tensors, in order.
 */
#define MI355_W8A8_FLAG_GRAD_TABLE_KEPT 1u
#define MI355_W8A8_GRAD_BF16 0u
#define MI355_W8A8_GRAD_F32 1u
#define MI355_W8A8_GRAD_MAX_TENSORS 65536u
typedef struct mi355_w8a8_grad_tensor {
  const void* grad;         /* [n_adapters, count], contiguous */
  void* out;                /* the same shape and type (mi355_w8a8_grad_norm_v1 ignores it) */
  uint64_t count;           /* values of one adapter; may be 0 */
  uint32_t type;            /* MI355_W8A8_GRAD_BF16 or _F32 */
  uint32_t reserved;        /* 0 */
} mi355_w8a8_grad_tensor;
uint64_t mi355_w8a8_grad_workspace_bytes(const mi355_w8a8_grad_tensor* tensors, uint32_t n_tensors, uint32_t n_adapters);
int mi355_w8a8_grad_norm_v1(const mi355_w8a8_grad_tensor* tensors, uint32_t n_tensors, uint32_t n_adapters, float* norms,
                            void* workspace, uint64_t workspace_bytes, uint32_t flags, void* stream);
int mi355_w8a8_grad_clip_v1(const mi355_w8a8_grad_tensor* tensors, uint32_t n_tensors, uint32_t n_adapters, const float* limits,
                            float* norms, void* workspace, uint64_t workspace_bytes, uint32_t flags, void* stream);

}  // extern "C"
