// The C entries of the dense layer.  linear.h holds the mathematics and the kernels; each type's are compiled in a translation unit of its own.
#include "linear.h"

namespace s2l {
namespace lin {

#define S2L_LINEAR_EXTERN(T)                                                                                                                  \
  extern template int forward<T>(Args, float*, hipStream_t);                                                                                  \
  extern template int backward<T>(const void*, int64_t, const void*, int64_t, const void*, int64_t, const void*, void*, int64_t, void*, void*, \
                                  char*, int64_t, int64_t, int64_t, int, float, hipStream_t);
S2L_LINEAR_EXTERN(float)
S2L_LINEAR_EXTERN(__bf16)
S2L_LINEAR_EXTERN(_Float16)

inline int size_of(int dtype) { return dtype == S2L_DTYPE_F32 ? 4 : dtype == S2L_DTYPE_BF16 || dtype == S2L_DTYPE_F16 ? 2 : 0; }
inline bool bad_dims(int64_t rows, int64_t in, int64_t out) {
  return rows < 0 || in < 1 || out < 1 || rows >= kMaxDim || in >= kMaxDim || out >= kMaxDim;
}
// elements lie on their own size; the workspace and what the library itself lays out there on 16 bytes
inline bool off(const void* p, int size) { return (reinterpret_cast<uintptr_t>(p) & (size - 1)) != 0; }

}  // namespace lin
}  // namespace s2l

extern "C" int64_t s2l_linear_saved_bytes(int dtype, int act, int64_t rows, int64_t out_features) {
  using namespace s2l::lin;
  if (!size_of(dtype) || bad_dims(rows, 1, out_features)) return 0;
  if (act == S2L_ACT_RELU || act == S2L_ACT_LEAKY_RELU) return rows * ((out_features + 7) >> 3);
  if (act == S2L_ACT_GELU || act == S2L_ACT_SILU) return rows * out_features * size_of(dtype);
  return 0;
}

extern "C" int64_t s2l_linear_forward_work_bytes(int dtype, int act, int keep, int64_t rows, int64_t in_features, int64_t out_features) {
  using namespace s2l::lin;
  if (!size_of(dtype) || bad_dims(rows, in_features, out_features) || skinny(rows, keep && (act == S2L_ACT_RELU || act == S2L_ACT_LEAKY_RELU))) return 0;
  return partial_bytes(plan_of(rows, out_features, in_features, size_of(dtype)), rows, out_features);
}

extern "C" int64_t s2l_linear_backward_work_bytes(int dtype, int act, int64_t rows, int64_t in_features, int64_t out_features) {
  using namespace s2l::lin;
  if (!size_of(dtype) || bad_dims(rows, in_features, out_features)) return 0;
  return back_plan(rows, in_features, out_features, size_of(dtype), act).total;
}

extern "C" int s2l_linear_forward(int dtype, const void* x, int64_t ldx, const void* weight, int64_t ldw, const void* bias, const void* residual, int64_t ldr, void* out,
                                  int64_t ldo, void* saved, void* work, int64_t rows, int64_t in_features, int64_t out_features, int act, float slope,
                                  s2l_stream_t stream) {
  using namespace s2l::lin;
  const int size = size_of(dtype);
  if (!size || act < S2L_ACT_NONE || act > S2L_ACT_SILU) return S2L_E_UNSUPPORTED;
  if (bad_dims(rows, in_features, out_features)) return S2L_E_SIZE;
  if (rows == 0) return S2L_OK;
  if (!x || !weight || !out) return S2L_E_NULL;
  if ((rows > 1 && (ldx < in_features || ldo < out_features || (residual && ldr < out_features))) || (out_features > 1 && ldw < in_features)) return S2L_E_SIZE;
  const int64_t need = s2l_linear_forward_work_bytes(dtype, act, saved != nullptr, rows, in_features, out_features);
  if (need && !work) return S2L_E_NULL;
  if (off(x, size) || off(weight, size) || off(bias, size) || off(residual, size) || off(out, size) || off(work, 16)) return S2L_E_ALIGN;
  const bool kinked = act == S2L_ACT_RELU || act == S2L_ACT_LEAKY_RELU, smooth = act == S2L_ACT_GELU || act == S2L_ACT_SILU;
  if (smooth && off(saved, size)) return S2L_E_ALIGN;
  Args g{};
  g.a = x;
  g.lda = ldx;
  g.b = weight;
  g.ldb = ldw;
  g.m = rows;
  g.n = out_features;
  g.k = in_features;
  g.bias = bias;
  g.residual = residual;
  g.ldr = ldr;
  g.out = out;
  g.ldo = ldo;
  g.act = act;
  g.slope = slope;
  g.bits = kinked ? static_cast<uint8_t*>(saved) : nullptr;
  g.zsave = smooth ? saved : nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  float* partial = static_cast<float*>(work);
  if (dtype == S2L_DTYPE_F32) return forward<float>(g, partial, st);
  if (dtype == S2L_DTYPE_BF16) return forward<__bf16>(g, partial, st);
  return forward<_Float16>(g, partial, st);
}

extern "C" int s2l_linear_backward(int dtype, const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* weight, int64_t ldw, const void* saved, void* dx,
                                   int64_t lddx, void* dweight, void* dbias, void* work, int64_t rows, int64_t in_features, int64_t out_features, int act, float slope,
                                   s2l_stream_t stream) {
  using namespace s2l::lin;
  const int size = size_of(dtype);
  if (!size || act < S2L_ACT_NONE || act > S2L_ACT_SILU) return S2L_E_UNSUPPORTED;
  if (bad_dims(rows, in_features, out_features)) return S2L_E_SIZE;
  if (dbias && !dweight) return S2L_E_NULL;      // the bias gradient is a by-product of dW
  if (!dx && !dweight) return S2L_OK;
  if (rows && (!dy || (act != S2L_ACT_NONE && !saved) || (dx && !weight) || (dweight && !x))) return S2L_E_NULL;
  if ((rows > 1 && (lddy < out_features || (dx && lddx < in_features) || (dweight && ldx < in_features))) || (dx && out_features > 1 && ldw < in_features)) return S2L_E_SIZE;
  const int64_t need = s2l_linear_backward_work_bytes(dtype, act, rows, in_features, out_features);
  if (need && !work) return S2L_E_NULL;
  if (off(dy, size) || off(x, size) || off(weight, size) || off(dx, size) || off(dweight, size) || off(dbias, size) || off(work, 16)) return S2L_E_ALIGN;
  if ((act == S2L_ACT_GELU || act == S2L_ACT_SILU) && off(saved, size)) return S2L_E_ALIGN;
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(work);
  if (dtype == S2L_DTYPE_F32)
    return backward<float>(dy, lddy, x, ldx, weight, ldw, saved, dx, lddx, dweight, dbias, ws, rows, in_features, out_features, act, slope, st);
  if (dtype == S2L_DTYPE_BF16)
    return backward<__bf16>(dy, lddy, x, ldx, weight, ldw, saved, dx, lddx, dweight, dbias, ws, rows, in_features, out_features, act, slope, st);
  return backward<_Float16>(dy, lddy, x, ldx, weight, ldw, saved, dx, lddx, dweight, dbias, ws, rows, in_features, out_features, act, slope, st);
}

extern "C" int s2l_debug_linear_routes(int dtype, int act, int keep, int grads, int64_t rows, int64_t in_features, int64_t out_features, int* routes) {
  using namespace s2l::lin;
  const int size = size_of(dtype);
  if (!size || act < S2L_ACT_NONE || act > S2L_ACT_SILU) return S2L_E_UNSUPPORTED;
  if (bad_dims(rows, in_features, out_features) || rows < 1) return S2L_E_SIZE;
  if (!routes) return S2L_E_NULL;
  const auto put = [&](int at, int path, int tile, int splits) {
    routes[at] = path;
    routes[at + 1] = tile;
    routes[at + 2] = splits;
  };
  const bool kinked = act == S2L_ACT_RELU || act == S2L_ACT_LEAKY_RELU;
  for (int i = 0; i < 10; ++i) routes[i] = 0;
  char* p = reinterpret_cast<char*>(uintptr_t{4096});      // (never read: an address of whole 16-byte pieces)
  if (skinny(rows, keep && kinked)) {
    put(0, 1, 0, 1);
  } else {
    Args g{};
    g.a = g.b = p;
    g.lda = g.ldb = g.k = in_features;
    g.m = rows;
    g.n = out_features;
    const Plan plan = plan_of(rows, out_features, in_features, size);
    const Route r = route_of(g, plan, true, true, size);
    put(0, r.dma ? 3 : 2, r.tile, plan.splits);
  }
  const Back b = back_plan(rows, in_features, out_features, size, act);
  const Products both = products_of(b, p, out_features, p, in_features, p, in_features, p, grads & 1 ? p : nullptr, in_features, grads & 2 ? p : nullptr, nullptr, rows,
                                    in_features, out_features, size, act, 0.5f);
  const Route dx = route_of(both.dx, b.dx, true, false, size), dw = route_of(both.dw, b.dw, false, false, size);
  if (grads & 1) put(3, both.together ? 4 : dx.dma ? 3 : 2, dx.tile, b.dx.splits);
  if (grads & 2) put(6, both.together ? 4 : dw.dma ? 3 : 2, dw.tile, b.dw.splits);
  routes[9] = !b.dz ? 0 : kinked ? 1 : b.slope.times;
  return S2L_OK;
}
