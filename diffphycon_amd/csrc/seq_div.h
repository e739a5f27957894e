// Division by a number the host knows: n / d for 0 <= n < 2^31 as (mulhi(n, m) + n) >> s with s = ceil(log2 d), m = floor(2^32 (2^s - d) / d) + 1.
#pragma once
#include "common.h"

namespace dpc {

struct Div {
    unsigned d, m, s;
    Div() : Div(1) {}
    explicit Div(unsigned x) : d(x), m(0), s(0) {
        while ((1ull << s) < d) ++s;
        m = (unsigned)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
    }
    __device__ __forceinline__ unsigned operator()(unsigned n) const { return (__umulhi(n, m) + n) >> s; }
    // n becomes n / d; returns n % d
    __device__ __forceinline__ int take(int& n) const {
        const int q = (int)(*this)((unsigned)n), r = n - q * (int)d;
        n = q;
        return r;
    }
};

}  // namespace dpc
