// What the two sources of the extension module _ncn_torch share.
#pragma once
#include <torch/extension.h>

namespace ncn_ext {

void check_status(const char* fn, int status);  // a non-zero status of the C ABI as the NCNError of _lib.py
bool plain(const at::Tensor& t);                // the memory is the value: no wrapper, no forward gradient
bool under_transform();                         // traced, or inside a functorch transform or a dispatch mode
void bind_attention(pybind11::module_& m);      // attn_torch.cpp

}  // namespace ncn_ext
