// Adds the block-norm functions of fln_torch_blocks.cpp to the extension module.
#pragma once
#include <torch/extension.h>

void fln_bind_blocks(pybind11::module& m);
