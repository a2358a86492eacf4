// A stand-in for what the adapter's decoder-layer classes use of the runtime
// (NodeProto, tensors, a context of named values, node helpers), of the GPU
// runtime (host memory) and of the library (calls that are written down, or
// refused as `refuse` says).  Test code: nothing here computes anything.
#pragma once
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <map>
#include <memory>
#include <mutex>
#include <stdexcept>
#include <string>
#include <unordered_set>
#include <utility>
#include <vector>

#include "onnxl_amd.h"

enum hipError_t { hipSuccess = 0 };
enum { hipMemcpyHostToDevice, hipMemcpyDeviceToHost };
inline int live_buffers = 0;
inline const char *hipGetErrorString(hipError_t) { return ""; }
inline hipError_t hipMalloc(void **p, size_t n) { *p = std::malloc(n); ++live_buffers; return hipSuccess; }
inline hipError_t hipFree(void *p) { std::free(p); --live_buffers; return hipSuccess; }
inline hipError_t hipMemcpy(void *d, const void *s, size_t n, int) { std::memcpy(d, s, n); return hipSuccess; }

struct NodeProto {
  std::string type;
  std::vector<std::string> in, out;
  std::map<std::string, int64_t> attributes;
  int input_size() const { return (int)in.size(); }
  int output_size() const { return (int)out.size(); }
  const std::string &input(int i) const { return in[i]; }
  const std::string &output(int i) const { return out[i]; }
  const std::string &op_type() const { return type; }
};

namespace rt {
struct Shape {
  std::vector<int64_t> d;
  Shape() = default;
  Shape(std::vector<int64_t> v) : d(std::move(v)) {}
  size_t size() const { return d.size(); }
  int64_t operator[](size_t i) const { return d[i]; }
};
struct Tensor {
  int32_t data_type = 0;
  Shape shape;
  std::vector<uint8_t> data;
  const uint8_t *bytes() const { return data.data(); }
  uint8_t *mutable_bytes() { return data.data(); }
  size_t size_bytes() const { return data.size(); }
};
struct RuntimeContext {
  std::map<std::string, Tensor> values;
  Tensor MakeOutputTensor(int, int32_t dt, Shape s, size_t n) { return Tensor{dt, std::move(s), std::vector<uint8_t>(n)}; }
  const Tensor &Get(const std::string &n) const { return values.at(n); }
};
struct KernelContext {
  const NodeProto *node;
};
struct KernelPreparationMemory {
  size_t a, b, c;
};
struct KernelPreparation {
  struct {
    std::vector<std::string> source_inputs;
    std::string representation;
    std::vector<std::string> output_slots;
  } info;
  std::function<KernelPreparationMemory(const RuntimeContext &)> estimate_memory;
  std::function<void(RuntimeContext &)> execute;
};
struct KernelBase {
  KernelBase(const KernelContext &k) : node_(k.node) {}
  virtual ~KernelBase() = default;
  virtual void Run(RuntimeContext &) = 0;
  virtual bool HasPreparations(const std::unordered_set<std::string> &) const { return false; }
  virtual void DeclarePreparations(const std::unordered_set<std::string> &, std::vector<KernelPreparation> &) {}
  const NodeProto *node_;
};
inline const Tensor *GetOptionalInput(const NodeProto &n, int i, RuntimeContext &c) {
  return i < n.input_size() && !n.input(i).empty() ? &c.values.at(n.input(i)) : nullptr;
}
inline int64_t GetAttributeIntOrDefault(const NodeProto &n, const char *name, int64_t d) {
  const auto it = n.attributes.find(name);
  return it == n.attributes.end() ? d : it->second;
}
inline void Require(bool ok) {
  if (!ok) throw std::invalid_argument("inputs or outputs");
}
inline void RequireMinInputCount(const NodeProto &n, int c) { Require(n.input_size() >= c); }
inline void RequireInputCount(const NodeProto &n, int c) { Require(n.input_size() == c); }
inline void RequireOutputCount(const NodeProto &n, int c) { Require(n.output_size() == c); }
inline void SetOutput(const NodeProto &n, int i, Tensor &&t, RuntimeContext &c) { c.values[n.output(i)] = std::move(t); }
inline size_t PackedByteSize(int32_t dt, int64_t n) {
  return dt == 1 || dt == 6 ? 4 * n : dt == 10 || dt == 16 ? 2 * n : dt == 23 ? (n + 1) / 2 : n;
}
}  // namespace rt

// ---- the library: every call is one line of what it was given ----------------
inline const char *refuse = nullptr;
inline void Put(const onnxl_amd_tensor *t) {
  if (t == nullptr || t->rank < 0) {
    std::printf(" -");
    return;
  }
  std::printf(" %d%s[", t->data_type, t->location == ONNXL_AMD_DEVICE ? "D" : "H");
  for (int i = 0; i < t->rank; ++i) std::printf(i ? ",%lld" : "%lld", (long long)t->dims[i]);
  std::printf("]%lld", (long long)t->size_bytes);
}
inline int Done() {
  std::printf("\n");
  return refuse ? ONNXL_AMD_INVALID_ARGUMENT : ONNXL_AMD_OK;
}
// a device tensor that the call changes
inline void Touch(onnxl_amd_tensor *t) { static_cast<uint8_t *>(t->data)[0] += 1; }
extern "C" {
inline const char *onnxl_amd_last_error() { return refuse; }
inline int onnxl_amd_synchronize(void *) { return ONNXL_AMD_OK; }
inline int onnxl_amd_rms_norm_quantize(const onnxl_amd_tensor *x, const onnxl_amd_tensor *w, const onnxl_amd_tensor *r,
                                       float eps, int64_t block, onnxl_amd_tensor *y, onnxl_amd_tensor *s,
                                       onnxl_amd_tensor *sum, void *) {
  std::printf("norm");
  for (auto *t : {x, w, r}) Put(t);
  std::printf(" %g %lld", eps, (long long)block);
  for (auto *t : {y, s, sum}) Put(t);
  return Done();
}
inline int onnxl_amd_mx_quantize(const onnxl_amd_tensor *x, onnxl_amd_tensor *y, onnxl_amd_tensor *s, void *) {
  std::printf("quantize");
  for (auto *t : {x, (const onnxl_amd_tensor *)y, (const onnxl_amd_tensor *)s}) Put(t);
  return Done();
}
inline int onnxl_amd_mx_matmul(const onnxl_amd_tensor *a, const onnxl_amd_tensor *as, int32_t a_type,
                               const onnxl_amd_tensor *b, const onnxl_amd_tensor *bs, onnxl_amd_tensor *y, void *) {
  std::printf("matmul");
  for (auto *t : {a, as}) Put(t);
  std::printf(" %d", a_type);
  for (auto *t : {b, bs, (const onnxl_amd_tensor *)y}) Put(t);
  return Done();
}
inline int onnxl_amd_kv_cache_append(const onnxl_amd_tensor *k, const onnxl_amd_tensor *v, onnxl_amd_tensor *kc,
                                     onnxl_amd_tensor *vc, onnxl_amd_tensor *ks, onnxl_amd_tensor *vs,
                                     const onnxl_amd_tensor *t, const onnxl_amd_tensor *s, const onnxl_amd_tensor *l,
                                     void *) {
  std::printf("append");
  for (const onnxl_amd_tensor *d : {k, v, (const onnxl_amd_tensor *)kc, (const onnxl_amd_tensor *)vc,
                                    (const onnxl_amd_tensor *)ks, (const onnxl_amd_tensor *)vs, t, s, l})
    Put(d);
  for (auto *d : {kc, vc, ks, vs}) Touch(d);
  return Done();
}
inline int onnxl_amd_kv_cache_attention(const onnxl_amd_tensor *q, const onnxl_amd_tensor *kc, const onnxl_amd_tensor *vc,
                                        const onnxl_amd_tensor *ks, const onnxl_amd_tensor *vs, const onnxl_amd_tensor *t,
                                        const onnxl_amd_tensor *s, const onnxl_amd_tensor *l, float scale,
                                        int64_t max_query, onnxl_amd_tensor *out, void *) {
  std::printf("attention");
  for (auto *d : {q, kc, vc, ks, vs, t, s, l}) Put(d);
  std::printf(" %g %lld", scale, (long long)max_query);
  Put(out);
  return Done();
}
}
