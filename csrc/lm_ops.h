// Registration of the operators around the language-model head (lm_ops.cpp).
#pragma once
#include <torch/extension.h>

void register_lm_ops(pybind11::module_& m);
