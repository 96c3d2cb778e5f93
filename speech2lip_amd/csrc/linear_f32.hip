// The dense layer's kernels on float (linear.h).
#include "linear.h"

namespace s2l {
namespace lin {
template int forward<float>(Args, float*, hipStream_t);
template int backward<float>(const void*, int64_t, const void*, int64_t, const void*, int64_t, const void*, void*, int64_t, void*, void*, char*, int64_t, int64_t,
                           int64_t, int, float, hipStream_t);
}  // namespace lin
}  // namespace s2l
