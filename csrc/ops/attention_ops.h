// Registers the attention operators with the extension module.
#pragma once

#include <pybind11/pybind11.h>

namespace bitscom_b200 {

void register_attention_bindings(pybind11::module_& m);

}  // namespace bitscom_b200
