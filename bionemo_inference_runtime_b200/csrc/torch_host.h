// What the parts of the native host path (_host.so) share.
#pragma once

#include <torch/extension.h>

#include <string>

namespace b200ta_host {

// Raises what _lib.call raises for a non-zero status of the entry point `fn`.
void check(int code, const char* fn);
std::string shape_of(const at::Tensor& t);

// torch_training.cpp: takes its entry points from the opened library, adds its functions to the module.
void bind_training(void* handle);
void define_training(pybind11::module_& m);

}  // namespace b200ta_host
