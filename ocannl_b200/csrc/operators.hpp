// Linked operators: what b200_layer_norm_link, b200_rotary_link, b200_attention_link and their gradients share.  An operator
// keeps the addresses its nodes have at link and a workspace of its own, as a linked routine does; a run only launches kernels
// on the device's stream.
#pragma once
#include <cuda_runtime.h>

#include <set>
#include <string>
#include <vector>

#include "runtime.hpp"

struct b200_operator {
  b200_dev* dev = nullptr;
  std::set<int> pools_used;      // what a run has to wait for, uploads-wise
  CUdeviceptr workspace = 0;
  size_t workspace_bytes = 0;
  virtual void run(cudaStream_t stream) = 0;
  virtual ~b200_operator() {}
  void take_workspace(size_t bytes) {
    workspace_bytes = bytes;
    if (!bytes) return;
    b200::cu_check(b200::cu().cuMemAlloc_(&workspace, bytes), "cuMemAlloc(operator workspace)");
  }
};

extern thread_local std::string b200_error_slot;  // api.cpp

namespace b200 {

inline size_t dtype_bytes(int dtype) { return dtype == B200_F32 ? 4 : 2; }

// Operands of one operator as byte ranges; outputs may overlap nothing else (but see `in_place`).
class Operands {
 public:
  Operands(b200_operator* op, const char* what) : op_(op), what_(what) {}
  [[noreturn]] void refuse(const std::string& why, int code = B200_E_INVALID) const { throw Error(code, std::string(what_) + ": " + why); }
  // `count` elements of `elem` bytes; 0 for an operand that is left out
  CUdeviceptr in(const b200_operand& o, const char* name, unsigned long long count, size_t elem, bool required = true) {
    return take(o, name, count, elem, required, false);
  }
  CUdeviceptr out(const b200_operand& o, const char* name, unsigned long long count, size_t elem, bool required = true) {
    return take(o, name, count, elem, required, true);
  }
  void dtype(int d) const {
    if (d != B200_F32 && d != B200_BF16 && d != B200_F16) refuse("unknown element type " + std::to_string(d));
  }
  // outputs that start at the same byte as an input of the same length are allowed where `in_place` names the pair
  void check_overlaps(const std::vector<std::pair<std::string, std::string>>& in_place = {}) const {
    for (size_t i = 0; i < all_.size(); ++i)
      for (size_t j = 0; j < all_.size(); ++j) {
        const Range &a = all_[i], &b = all_[j];
        if (i == j || !a.written || (b.written && j < i)) continue;
        if (a.end <= b.begin || b.end <= a.begin) continue;
        bool ok = false;
        for (auto& p : in_place) ok |= p.first == a.name && p.second == b.name && a.begin == b.begin && a.end == b.end;
        if (!ok) refuse("the output '" + a.name + "' overlaps '" + b.name + "'");
      }
  }

 private:
  struct Range {
    std::string name;
    CUdeviceptr begin, end;
    bool written;
  };
  CUdeviceptr take(const b200_operand& o, const char* name, unsigned long long count, size_t elem, bool required, bool written) {
    if (o.pool_id < 0) {
      if (required) refuse(std::string("'") + name + "' is required");
      return 0;
    }
    if (o.offset % elem) refuse(std::string("'") + name + "' is bound at offset " + std::to_string(o.offset) + ", not a multiple of its element size");
    const unsigned __int128 bytes = (unsigned __int128)count * elem;
    if (bytes >> 62) refuse(std::string("'") + name + "' is too large");
    const CUdeviceptr p = op_->dev->address(o.pool_id, (size_t)o.offset, (size_t)bytes);
    op_->pools_used.insert(o.pool_id);
    if (bytes) all_.push_back({name, p, p + (CUdeviceptr)bytes, written});
    return p;
  }
  b200_operator* op_;
  const char* what_;
  std::vector<Range> all_;
};

// a * b * .. of extents, refused where it passes 2^62
inline unsigned long long extent_product(std::initializer_list<long long> v, const char* what) {
  unsigned __int128 p = 1;
  for (long long x : v) {
    if (x < 0) throw Error(B200_E_INVALID, std::string(what) + ": negative extent");
    p *= (unsigned long long)x;
    if (p >> 62) throw Error(B200_E_INVALID, std::string(what) + ": too many elements");
  }
  return (unsigned long long)p;
}

inline void rt_check(cudaError_t e, const char* what) {
  if (e != cudaSuccess) throw Error((int)e, std::string(what) + ": " + cudaGetErrorString(e));
}

// launches of operators on this thread, for the device's count (api.cpp)
inline thread_local long long operator_launches = 0;

// Programmatic stream serialisation, as every launch of the library: the kernels release their dependents at entry and wait
// for the grids ahead before they touch memory.
template <class... P, class... A>
void launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  rt_check(cudaLaunchKernelEx(&cfg, kernel, P(args)...), "operator launch");
  ++operator_launches;
}

// Loads a kernel's code now (nothing is loaded inside a run, which may be under capture) and allows it its shared memory.
template <class K>
void ready(K kernel, size_t smem = 0) {
  cudaFuncAttributes a;
  rt_check(cudaFuncGetAttributes(&a, kernel), "cudaFuncGetAttributes");
  // (never lowered: operators that were linked before may need more)
  if ((int)smem > a.maxDynamicSharedSizeBytes) rt_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "cudaFuncSetAttribute");
}

// The body of a link entry point: `make` fills a new operator of class Op; nothing crosses the C boundary.
template <class Op, class F>
int link_operator(b200_dev* dev, const void* spec, b200_operator** out, F&& make) {
  Op* op = nullptr;
  try {
    if (!dev || !spec || !out) throw Error(B200_E_INVALID, "null argument");
    *out = nullptr;
    dev->make_current();
    op = new Op();
    op->dev = dev;
    make(op);
    *out = op;
    return 0;
  } catch (const Error& e) {
    b200_error_slot = e.what();
    if (op && op->workspace) cu().cuMemFree_(op->workspace);
    delete op;
    return e.code;
  } catch (const std::exception& e) {
    b200_error_slot = e.what();
    if (op && op->workspace) cu().cuMemFree_(op->workspace);
    delete op;
    return B200_E_INVALID;
  }
}

}  // namespace b200
