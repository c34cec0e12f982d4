// Whether two strided arrays may share memory (host only): what a kernel writes must not be what other threads of it still read.
#pragma once
#include <cstdint>
#include <initializer_list>

namespace amp {

struct SpanDim { long size, stride; };         // stride in bytes

struct Span
{
    uintptr_t at;                              // first byte
    long inner;                                // bytes without a gap
    int n = 0;
    SpanDim dim[4];                            // without those of one place, and broadcast ones

    Span(const void* p, long bytes, std::initializer_list<SpanDim> dims) : at((uintptr_t) p), inner(bytes)
    {
        for (SpanDim d : dims)
        {
            if (d.size <= 1 || d.stride == 0) continue;
            if (d.stride < 0) { at += (d.size - 1) * d.stride; d.stride = -d.stride; }
            dim[n++] = d;
        }
    }
    // bytes from the first to behind the last one, counted round `period` (0: not at all)
    long extent(long period) const
    {
        long e = inner;
        for (int i = 0; i < n; ++i) if (!period || dim[i].stride % period) e += (dim[i].size - 1) * dim[i].stride;
        return e;
    }
    bool same(const Span& o) const
    {
        bool s = at == o.at && inner == o.inner && n == o.n;
        for (int i = 0; s && i < n; ++i) s = dim[i].size == o.dim[i].size && dim[i].stride == o.dim[i].stride;
        return s;
    }
};

// No byte of a is one of b: their extents lie apart, or they do round one of their strides (columns of one buffer, keys and values side by side
// in a page, every other row). Arrays that share nothing in a more tangled way count as sharing.
inline bool apart(const Span& a, const Span& b)
{
    if (a.at + a.extent(0) <= b.at || b.at + b.extent(0) <= a.at) return true;
    for (const Span* s : { &a, &b })
        for (int i = 0; i < s->n; ++i)
        {
            const long p = s->dim[i].stride, ea = a.extent(p), eb = b.extent(p);
            if (ea > p || eb > p) continue;
            const long d = (long) (b.at >= a.at ? (b.at - a.at) % p : (p - (a.at - b.at) % p) % p);
            if (d >= ea && d + eb <= p) return true;
        }
    return false;
}

}  // namespace amp
