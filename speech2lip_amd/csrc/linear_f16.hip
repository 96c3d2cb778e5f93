// The dense layer's kernels on _Float16 (linear.h).
#include "linear.h"

namespace s2l {
namespace lin {
template int forward<_Float16>(Args, float*, hipStream_t);
template int backward<_Float16>(const void*, int64_t, const void*, int64_t, const void*, int64_t, const void*, void*, int64_t, void*, void*, char*, int64_t, int64_t,
                           int64_t, int, float, hipStream_t);
}  // namespace lin
}  // namespace s2l
