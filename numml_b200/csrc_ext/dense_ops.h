// The dense operators of the graph layers as functions of the compiled extension.
#pragma once
#include <torch/extension.h>

void register_dense_ops(py::module_& m);
