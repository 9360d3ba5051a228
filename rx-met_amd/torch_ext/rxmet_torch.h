// rxmet_torch.h — what the sources of the module rxmet_torch share.
#pragma once

#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <stdexcept>
#include <string>

namespace rxmet_torch {

// A failing call of the library: rxmet_lib.RxmetError in Python.
struct LibraryError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

inline void *stream_of(const at::Tensor &t) {
  return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

// decoder_torch.cpp
void add_decoder(pybind11::module_ &m);
// expert_torch.cpp
void add_experts(pybind11::module_ &m);

}  // namespace rxmet_torch
