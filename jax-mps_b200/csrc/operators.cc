// Dispatch of the operators that programs name as custom calls.
#include "operators.h"

namespace b200 {

bool operators_programmatic_launch = true;
void set_operators_programmatic_launch(bool on) { operators_programmatic_launch = on; }

const char* operator_plan(OperatorLaunch& op) {
  switch (op.kind) {
    case OperatorLaunch::PAGED_ATTENTION: return paged_attention_plan(op);
    case OperatorLaunch::WINDOW_ATTENTION: return window_attention_plan(op);
    case OperatorLaunch::TOKEN_LOG_PROBS: case OperatorLaunch::TOKEN_LOG_PROBS_GRAD: case OperatorLaunch::TOKEN_LOG_PROBS_BOTH: return token_log_probs_plan(op);
    default: return "no operator";
  }
}

cudaError_t launch_operator(const OperatorLaunch& op, void* const* args, void* scratch, int* error_flag, cudaStream_t stream, int* launches, const char** why) {
  switch (op.kind) {
    case OperatorLaunch::PAGED_ATTENTION: return launch_paged_attention(op, args, scratch, stream, launches);
    case OperatorLaunch::WINDOW_ATTENTION: return launch_window_attention(op, args, scratch, error_flag, stream, launches, why);
    case OperatorLaunch::TOKEN_LOG_PROBS: return launch_token_log_probs(op, args, scratch, stream, launches);
    case OperatorLaunch::TOKEN_LOG_PROBS_BOTH: return launch_token_log_probs_both(op, args, stream, launches);
    case OperatorLaunch::TOKEN_LOG_PROBS_GRAD: return launch_token_log_probs_grad(op, args, stream, launches);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace b200
