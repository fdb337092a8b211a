// afa_torch_common.h -- what the two source files of the torch extension share:
// the per-device status word and the checks every entry point makes.
#pragma once

#include <torch/extension.h>

#include <cstdint>

namespace afa_torch {

#define AFA_CHECK_CUDA(x) TORCH_CHECK((x).device().is_cuda(), #x " must be a CUDA tensor")
#define AFA_CHECK_LAST_DIM(x) \
  TORCH_CHECK((x).dim() == 4 && (x).stride(3) == 1, #x " must be 4-D [batch, seq, heads, head_dim] with a contiguous head_dim")

// AFA_DTYPE_* of a tensor, -1 for other types.
int dtype_code(const at::Tensor& t);

// One status word per device (int32, zero = ok) in mapped page-locked host
// memory: every launch on the device gets its device address, a kernel whose
// bounded wait runs out (or, in the cache operators, that meets a bad page or
// length) stores its code there, and the host reads it without synchronising.
// Each call first takes (and clears) what earlier launches on its device
// reported, so a device-side abort is raised by the next call on that device --
// at the latest by the first one made after the aborted launch has finished --
// or by check_status(), which synchronises first.  Kept until the process exits
// (4 bytes of page-locked memory per device).
struct StatusWord {
  int32_t* host = nullptr;    // what the host reads
  int32_t* device = nullptr;  // the same word as the kernel addresses it
};
StatusWord status_word(int dev);

// Takes the code earlier launches on `dev` left in the status word and clears it.
int32_t take_status(int dev);

// Raises for an abort that a launch made before this call reported.
void raise_earlier_abort(int dev);

// Adds the operators of afa_torch_ops.cpp to the module.
void bind_ops(pybind11::module_& m);

}  // namespace afa_torch
