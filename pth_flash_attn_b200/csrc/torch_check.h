// What the op files of the paged caches share: argument checks that name their argument, the device's stream, and the C ABI's
// argument structs.
#pragma once

#include <cuda_runtime.h>
#include <torch/csrc/stable/accelerator.h>
#include <torch/csrc/stable/library.h>
#include <torch/csrc/stable/tensor.h>
#include <torch/headeronly/core/ScalarType.h>
#include <torch/headeronly/util/Exception.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <utility>

#include "../../include/pthb200_attn.h"

extern "C" int32_t aoti_torch_get_current_cuda_stream(int32_t device_index, void** ret_stream);

namespace {

using torch::headeronly::ScalarType;
using torch::stable::Tensor;

const char* type_name(ScalarType t) {
  switch (t) {
    case ScalarType::BFloat16: return "bfloat16";
    case ScalarType::Half: return "float16";
    case ScalarType::Float: return "float32";
    case ScalarType::Byte: return "uint8";
    case ScalarType::Char: return "int8";
    case ScalarType::Int: return "int32";
    case ScalarType::Long: return "int64";
    case ScalarType::Double: return "float64";
    case ScalarType::Float8_e4m3fn: return "float8_e4m3fn";
    default: return "an unsupported dtype";
  }
}
int32_t type_code(ScalarType t) {
  return t == ScalarType::Float ? PTH_ATTN_F32 : t == ScalarType::Half ? PTH_ATTN_F16 : PTH_ATTN_BF16;
}

struct Check {
  const char* op;  // "name: ", the start of every message

  void rank(const Tensor& t, int64_t want, const char* name) const {
    STD_TORCH_CHECK(t.dim() == want, op, name, " must be ", want, "-D, got ", t.dim(), "-D");
  }
  void dtype(const Tensor& t, ScalarType want, const char* name) const {
    STD_TORCH_CHECK(t.scalar_type() == want, op, name, " must be ", type_name(want), ", got ", type_name(t.scalar_type()));
  }
  void size(const Tensor& t, int64_t dim, int64_t want, const char* name, const char* what) const {
    STD_TORCH_CHECK(t.size(dim) == want, op, name, ".size(", dim, ") must equal ", what, " = ", want, ", got ", t.size(dim));
  }
  void inner(const Tensor& t, const char* name) const {
    STD_TORCH_CHECK(t.numel() == 0 || t.stride(t.dim() - 1) == 1, op, name, " must have stride 1 in its last dimension, got ",
                    t.stride(t.dim() - 1));
  }
  // of a tensor that the op writes: every element has a place of its own, as far as strides of zero go
  void written(const Tensor& t, const char* name) const {
    for (int64_t d = 0; d < t.dim(); ++d)
      STD_TORCH_CHECK(t.size(d) <= 1 || t.stride(d) != 0 || t.numel() == 0, op, name, " is written and must not have stride 0, as in dimension ", d);
  }
  void device(const Tensor& t, const Tensor& as, const char* name, const char* of) const {
    // (a CPU tensor's index is -1)
    STD_TORCH_CHECK(t.get_device_index() == as.get_device_index(), op, name, " must be on the same device as ", of);
  }
  void vector(const Tensor& t, ScalarType type, const char* name) const {
    rank(t, 1, name);
    dtype(t, type, name);
    inner(t, name);
  }
  // a size that the C ABI carries in 32 bits
  void count(int64_t n, const char* name) const {
    STD_TORCH_CHECK(n >= 0 && n <= INT32_MAX, op, name, " = ", n, " is out of range");
  }
  // Where the arguments are in order: the device's stream (raises for tensors of another device).
  void* stream(const Tensor& t, int32_t* index) const {
    STD_TORCH_CHECK(t.is_cuda(), op,
                    "arguments are valid, but the op computes on CUDA tensors only (the CPU registration exists to test the "
                    "argument checks)");
    *index = static_cast<int32_t>(t.get_device_index());
    int major = 0;
    const cudaError_t err = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, *index);
    STD_TORCH_CHECK(err == cudaSuccess, op, "cannot query the compute capability: ", cudaGetErrorString(err));
    STD_TORCH_CHECK(major == 10, op, "needs compute capability 10.x (sm_100a), device has major ", major);
    void* s = nullptr;
    STD_TORCH_CHECK(aoti_torch_get_current_cuda_stream(*index, &s) == 0, op, "cannot get the current CUDA stream of device ", *index);
    return s;
  }
  void done(int32_t rc) const { STD_TORCH_CHECK(rc == PTH_ATTN_OK, op, pthb200_last_error()); }
};

int64_t bytes(const Tensor& t, int64_t dim) { return t.stride(dim) * static_cast<int64_t>(t.element_size()); }
PthAttnStream as_stream(const Tensor& t) { return PthAttnStream{t.data_ptr(), bytes(t, 0), bytes(t, 1), bytes(t, 2)}; }
template <class Args>
Args new_args() {
  Args a{};
  a.abi_version = PTH_ATTN_ABI_VERSION;
  a.struct_bytes = static_cast<int32_t>(sizeof(Args));
  return a;
}

}  // namespace
