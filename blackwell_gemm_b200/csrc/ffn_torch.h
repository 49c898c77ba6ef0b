// Torch bindings of the feed-forward operators; registered by the extension's
// module definition in matmul.cpp.
#pragma once
#include <torch/extension.h>

void register_ffn(pybind11::module_& m);
