// The library's part of adapter_runtime.hpp for the operators from a layer's joint
// projection to the next token: every call is one line of what it was given.
#pragma once
#include "adapter_runtime.hpp"

extern "C" {
inline int onnxl_amd_mx_gated_matmul(const onnxl_amd_tensor *a, const onnxl_amd_tensor *as, int32_t a_type,
                                     const onnxl_amd_tensor *g, const onnxl_amd_tensor *gs, const onnxl_amd_tensor *u,
                                     const onnxl_amd_tensor *us, int32_t activation, onnxl_amd_tensor *y,
                                     onnxl_amd_tensor *ys, void *) {
  std::printf("gated");
  for (auto *t : {a, as}) Put(t);
  std::printf(" %d", a_type);
  for (auto *t : {g, gs, u, us}) Put(t);
  std::printf(" %d", activation);
  for (auto *t : {y, ys}) Put(t);
  return Done();
}
inline int onnxl_amd_rotary_tables(double base, int32_t scaling, double factor, int64_t original, double fast, double slow,
                                   double magnitude, onnxl_amd_tensor *c, onnxl_amd_tensor *s, void *) {
  std::printf("tables %g %d %g %lld %g %g %g", base, scaling, factor, (long long)original, fast, slow, magnitude);
  for (auto *t : {c, s}) Put(t);
  return Done();
}
inline int onnxl_amd_rotary_embedding(const onnxl_amd_tensor *x, const onnxl_amd_tensor *c, const onnxl_amd_tensor *s,
                                      const onnxl_amd_tensor *ids, int32_t interleaved, int64_t heads, onnxl_amd_tensor *y,
                                      void *) {
  std::printf("rotary");
  for (auto *t : {x, c, s, ids}) Put(t);
  std::printf(" %d %lld", interleaved, (long long)heads);
  Put(y);
  return Done();
}
inline int onnxl_amd_rotary_kv_cache_append(const onnxl_amd_tensor *x, const onnxl_amd_tensor *c, const onnxl_amd_tensor *s,
                                            const onnxl_amd_tensor *ids, int32_t interleaved, onnxl_amd_tensor *q,
                                            onnxl_amd_tensor *kc, onnxl_amd_tensor *vc, onnxl_amd_tensor *ks,
                                            onnxl_amd_tensor *vs, const onnxl_amd_tensor *t, const onnxl_amd_tensor *st,
                                            const onnxl_amd_tensor *l, void *) {
  std::printf("rotary append");
  for (auto *d : {x, c, s, ids}) Put(d);
  std::printf(" %d", interleaved);
  for (const onnxl_amd_tensor *d : {(const onnxl_amd_tensor *)q, (const onnxl_amd_tensor *)kc, (const onnxl_amd_tensor *)vc,
                                    (const onnxl_amd_tensor *)ks, (const onnxl_amd_tensor *)vs, t, st, l})
    Put(d);
  for (auto *d : {q, kc, vc, ks, vs}) Touch(d);
  return Done();
}
inline int onnxl_amd_sample_tokens(const onnxl_amd_tensor *x, const onnxl_amd_tensor *u, const onnxl_amd_tensor *t,
                                   const onnxl_amd_tensor *k, const onnxl_amd_tensor *p, const onnxl_amd_tensor *m,
                                   onnxl_amd_tensor *token, onnxl_amd_tensor *prob, void *) {
  std::printf("sample");
  for (auto *d : {x, u, t, k, p, m, (const onnxl_amd_tensor *)token, (const onnxl_amd_tensor *)prob}) Put(d);
  return Done();
}
}
