// Registration hook that lets further binding files add functions to the one extension module.
#pragma once
#include <pybind11/pybind11.h>
void sg_register_extra(pybind11::module_& m);
void sg_register_device_io(pybind11::module_& m);  // device_file_io.cpp
void sg_register_decode(pybind11::module_& m);     // bindings_decode.cpp
// Adds n to the extension-wide count of kernels launched (read through launch_count()).
void sg_count_launch(int n);
// The current device's int32 word that kernels set when something went wrong.
int* sg_error_flag();
