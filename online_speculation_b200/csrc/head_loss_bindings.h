// Registers the bindings of head_loss_bindings.cpp with the extension module.
#pragma once
#include <pybind11/pybind11.h>

void register_head_losses(pybind11::module_& m);
