// Arguments of the tensor-core kernels over a paged cache (paged_tc.cu), as their callers fill them.
#pragma once
#include "serving_plan.cuh"

namespace risa_b200 {
namespace serving {

constexpr int kTcWorkers = 148;  // one CTA per SM
// Sequences with at least so many query rows per key head are theirs.
constexpr int kTcFewestRows = 33;

struct TcArgs {
  LineArgs line;  // rows, keys and notes are the kernel's own: paged_tc_args
  const void* q;
  int64_t qn, qh;
  void* out;
  int64_t on, oh;
  float* lse;
  const char* keys;
  const char* values;
  const float* key_scales;
  const float* value_scales;
  int pages;
  float scale_log2;
  float* parts;
  JoinNote* notes;  // behind the parts
  int min_steps;
  unsigned int* status;
};

size_t paged_tc_scratch(int head_dim);
// The kernel runs beside the launch in front of it, which has to be one of the same call that succeeded; the join comes behind both.
TcArgs paged_tc_args(TcArgs args, int head_dim);
int paged_tc(const TcArgs& args, int dtype_code, bool codes, int head_dim, cudaStream_t stream);
int paged_tc_join(const TcArgs& args, int dtype_code, int head_dim, cudaStream_t stream);
int paged_tc_wait_status();

// Key weights (weigh_tc.cu), likewise beside the launch in front; `out`, `lse` and `values` of the arguments are not used.
size_t weigh_tc_scratch();
int weigh_tc(const TcArgs& args, const float* row_lse, const float* previous, float* weights, int dtype_code, bool codes, int head_dim,
             cudaStream_t stream);
int weigh_tc_wait_status();

}  // namespace serving
}  // namespace risa_b200
