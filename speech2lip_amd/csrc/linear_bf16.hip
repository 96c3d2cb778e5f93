// The dense layer's kernels on __bf16 (linear.h).
#include "linear.h"

namespace s2l {
namespace lin {
template int forward<__bf16>(Args, float*, hipStream_t);
template int backward<__bf16>(const void*, int64_t, const void*, int64_t, const void*, int64_t, const void*, void*, int64_t, void*, void*, char*, int64_t, int64_t,
                           int64_t, int, float, hipStream_t);
}  // namespace lin
}  // namespace s2l
