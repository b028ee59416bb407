// Shared by the sources of the torch binding (_trring_torch).
#pragma once

#include <pybind11/pybind11.h>
#include <torch/extension.h>

#include <stdexcept>
#include <string>

#include "trring.h"

namespace trr_torch {

// TR_ERR_INVALID becomes ValueError, every other status RuntimeError
[[noreturn]] inline void raise_status(int st, const char* what) {
  std::string msg = std::string(what) + ": " + tr_status_string(st) + " (" + tr_last_error() + ")";
  if (st == TR_ERR_INVALID) throw pybind11::value_error(msg);
  throw std::runtime_error(msg);
}

inline int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return TR_F32;
    case at::kHalf: return TR_F16;
    case at::kBFloat16: return TR_BF16;
    default: return -1;
  }
}

void bind_serving(pybind11::module_& m);  // torch_serve.cpp

}  // namespace trr_torch
