// Torch bindings of the mixture-of-experts operators; registered by the
// extension's module definition in matmul.cpp.
#pragma once
#include <torch/extension.h>

void register_moe(pybind11::module_& m);
