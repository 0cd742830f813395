// fa_ops.h - the operators that fa_ops.cpp adds to the module of fa_autograd.cpp.
#pragma once

#include <pybind11/pybind11.h>

void fa_def_ops(pybind11::module_& m);
