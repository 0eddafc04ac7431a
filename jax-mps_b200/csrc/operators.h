// Operators of large language models that a program names as custom calls (`stablehlo.custom_call @b200.<name>`), and the moves
// inside a paged cache that the client offers beside them. One launch description for the plan compiler, which fills and sizes
// it, and the launchers, which follow it.
#pragma once
#include <cuda_runtime.h>

namespace b200 {

struct OperatorLaunch {
  enum Kind { NONE, PAGED_ATTENTION, WINDOW_ATTENTION, TOKEN_LOG_PROBS, TOKEN_LOG_PROBS_GRAD, TOKEN_LOG_PROBS_BOTH } kind = NONE;
  int type = 0;                             // of the data: 0 f32, 1 bf16, 2 f16
  // attention: sequences, tokens of each (prompt), query and key-value heads, features of a head
  int batch = 0, tokens = 0, heads = 0, kv_heads = 0, dim = 0;
  int window = 0, sinks = 0;                // 0: no window
  float scale = 1.f;
  // cache [layers, 2, pages, page, kv_heads, dim], of which one layer is read through a table of `width` pages per sequence
  int layer = 0, pages = 0, page = 1, width = 0;
  int has_new = 0, has_lengths = 1;
  // log probabilities: rows of `vocab` logits, the best `top` of each
  long long rows = 0;
  int vocab = 0, top = 0;
  // filled by operator_plan
  long long scratch_bytes = 0;
  int launches = 0;
  int waits = 0;                            // a kernel has bounded waits: executions read the error word back
};

// Chooses kernels and sizes the scratch memory; null, or why the operator cannot run.
const char* operator_plan(OperatorLaunch& op);
void set_operators_programmatic_launch(bool on);
// `args`: results, then operands, in the order of the custom call.
cudaError_t launch_operator(const OperatorLaunch& op, void* const* args, void* scratch, int* error_flag, cudaStream_t stream, int* launches, const char** why);

// One per kernel file.
const char* paged_attention_plan(OperatorLaunch& op);
cudaError_t launch_paged_attention(const OperatorLaunch& op, void* const* args, void* scratch, cudaStream_t stream, int* launches);
const char* window_attention_plan(OperatorLaunch& op);
cudaError_t launch_window_attention(const OperatorLaunch& op, void* const* args, void* scratch, int* error_flag, cudaStream_t stream, int* launches, const char** why);
const char* token_log_probs_plan(OperatorLaunch& op);
cudaError_t launch_token_log_probs(const OperatorLaunch& op, void* const* args, void* scratch, cudaStream_t stream, int* launches);
// Log probabilities and their gradient by one reading of the logits: results, gradient, logits, tokens, the three cotangents.
bool token_log_probs_at_once(const OperatorLaunch& op);
cudaError_t launch_token_log_probs_both(const OperatorLaunch& op, void* const* args, cudaStream_t stream, int* launches);
cudaError_t launch_token_log_probs_grad(const OperatorLaunch& op, void* const* args, cudaStream_t stream, int* launches);

// Moves inside a cache. `token`: bytes of one token's keys (or values) of one layer; planes = layers * 2. The index arrays are
// host memory, read before the call returns, and have been checked by the caller.
struct CacheShape {
  long long planes, pages, page, token;
};
cudaError_t launch_write_pages(const CacheShape& c, void* cache, const void* rows, const int* slots, long long n, cudaStream_t stream, int* launches);
// Pairs are (source, destination). The source of pair i is read from place staged[i] of `stage` where that is not negative.
cudaError_t launch_copy_pages(const CacheShape& c, void* cache, const int* pairs, const int* staged, const void* stage, long long n, cudaStream_t stream, int* launches);
// Copies page sources[i] of every plane to place i of `stage`.
cudaError_t launch_stage_pages(const CacheShape& c, const void* cache, void* stage, const int* sources, long long n, cudaStream_t stream, int* launches);

}  // namespace b200
