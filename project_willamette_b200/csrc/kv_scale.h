// kv_scale.h -- how the scale of a page of the paged int8 KV cache grows when a
// call appends rows behind others.  Plain C++, so that it is checked without a GPU.
#pragma once

#include <cmath>

#ifdef __CUDACC__
#define WL_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define WL_HOST_DEVICE inline
#endif

namespace wl {

// The smallest float that is not 0, 2^-149, reaches the largest need, below 2^122, in so
// many doublings.
constexpr int PAGE_SCALE_MAX_DOUBLINGS = 271;

struct PageScale {
    float scale;
    int doublings;
};

// `old` is the page's scale, `need` (>= 0 or NaN) the largest |new value| / 127.  A page that
// other code filled may have a negative scale (a code c stands for c * scale all the same):
// its size grows and it keeps its sign.  NaN and infinities stay.
WL_HOST_DEVICE PageScale grown_scale(float old, float need) {
    PageScale g = {old, 0};
    if (need != need || old == 0.0f) {
        g.scale = need;
    } else {
        while (fabsf(g.scale) < need && g.doublings < PAGE_SCALE_MAX_DOUBLINGS) {
            g.scale *= 2.0f;
            ++g.doublings;
        }
    }
    return g;
}

}  // namespace wl
