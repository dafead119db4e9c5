// operators.h -- the model head's launches (include/flashtrie_amd.h), between
// the argument checks (operators.cpp) and the kernels.
#ifndef FTAMD_OPERATORS_H_
#define FTAMD_OPERATORS_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/flashtrie_amd.h"

namespace fto {

inline uint64_t round_up(uint64_t v, uint64_t a) { return (v + a - 1) / a * a; }

// Parts of a workspace, each 256-byte aligned.
struct Arena {
  uint64_t used = 0;
  uint64_t take(uint64_t bytes) {
    const uint64_t at = used;
    used = round_up(used + bytes, 256);
    return at;
  }
};

// Starts a kernel of one argument.  The launch's own status: the runtime's
// last error may be that of another call of the application.
template <typename A>
hipError_t start(void (*kernel)(A), uint64_t blocks, uint32_t threads, hipStream_t s, A a) {
  void* args[] = {&a};
  const hipError_t e = hipLaunchKernel((const void*)kernel, dim3((uint32_t)blocks), dim3(threads),
                                       args, 0, s);
  if (e != hipSuccess) (void)hipGetLastError();  // it is in the caller's hands now
  return e;
}

uint64_t adapter_logits_workspace(const ft_adapter_logits_args& a);
hipError_t launch_adapter_logits(const ft_adapter_logits_args& a, uint8_t* ws, hipStream_t s);

uint64_t propose_workspace(const ft_propose_args& a);
hipError_t launch_propose(const ft_propose_args& a, uint8_t* ws, hipStream_t s);

uint64_t policy_loss_workspace(const ft_policy_loss_args& a);
hipError_t launch_policy_loss(const ft_policy_loss_args& a, uint8_t* ws, hipStream_t s);

uint64_t preference_loss_workspace(const ft_preference_loss_args& a);
hipError_t launch_preference_loss(const ft_preference_loss_args& a, uint8_t* ws, hipStream_t s);

uint64_t cross_entropy_loss_workspace(const ft_cross_entropy_loss_args& a);
hipError_t launch_cross_entropy_loss(const ft_cross_entropy_loss_args& a, uint8_t* ws, hipStream_t s);

uint64_t pack_weight_workspace(const ft_pack_weight_args& a);
hipError_t launch_pack_weight(const ft_pack_weight_args& a, uint8_t* ws, hipStream_t s);

uint64_t packed_logits_workspace(const ft_packed_logits_args& a);
hipError_t launch_packed_logits(const ft_packed_logits_args& a, uint8_t* ws, hipStream_t s);

uint64_t embed_workspace(const ft_embed_args& a);
hipError_t launch_embed(const ft_embed_args& a, uint8_t* ws, hipStream_t s);

uint64_t embed_grad_workspace(const ft_embed_grad_args& a);
hipError_t launch_embed_grad(const ft_embed_grad_args& a, uint8_t* ws, hipStream_t s);

}  // namespace fto

namespace ftk {
// the text behind ft_last_error, and the code back (ft_runtime.cpp)
int set_error(int code, const char* msg) noexcept;
}  // namespace ftk

#endif  // FTAMD_OPERATORS_H_
