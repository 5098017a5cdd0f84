// What the translation units of the host module share.
#pragma once
#include <Python.h>

#include <string>

#include <ATen/ATen.h>

namespace mvr_host {

std::string type_name(at::ScalarType t);  // as Python spells it
int label_type(at::ScalarType t);         // MVR_LABEL_*, or -1
void check(int rc);                       // throws what the library's code means
int* status_of(int device);               // the device's status word

PyMethodDef* head_methods();              // functions of mvr_torch_heads.cpp

}  // namespace mvr_host
