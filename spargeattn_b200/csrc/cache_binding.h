// Functions of cache_binding.cpp that binding.cpp adds to its module, and what it gives them.
#pragma once
#include <Python.h>

#include <ATen/ATen.h>

extern PyMethodDef kCacheMethods[];

// The int32 word of a device that kernels report to, or null before one is registered.
at::Tensor* cache_status_word(int device);
