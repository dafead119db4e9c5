// bind_operators.h -- adds the model head's operators to the Python module.
#ifndef FTAMD_BIND_OPERATORS_H_
#define FTAMD_BIND_OPERATORS_H_

#include <pybind11/pybind11.h>

void bind_operators(pybind11::module_& m);

#endif  // FTAMD_BIND_OPERATORS_H_
