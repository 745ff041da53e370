// What tccl_host_ops.cpp adds to the extension module of tccl_host.cpp.
#pragma once

#include <Python.h>

PyMethodDef* operator_methods();
