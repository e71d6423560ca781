// Whether two tensors that a caller describes share memory (host code).
#pragma once
#include <stdint.h>
#include <algorithm>
#include <utility>

// A tensor [B][T][width] as a caller describes it.
struct StesRows {
    const void* p;
    int es;                 // bytes of an element
    int64_t ld, bs;         // elements between frames, between sequences
    int64_t T, B, width;
};

static inline bool stes_share(StesRows a, StesRows b) {
    if (!a.p || !b.p || !a.T || !a.B || !a.width || !b.T || !b.B || !b.width) return false;
    auto span = [](const StesRows& r) { return (r.T - 1) * r.ld + r.width; };
    auto bytes = [&](const StesRows& r) { return ((r.B - 1) * r.bs + span(r)) * r.es; };
    const int64_t d = (const char*)b.p - (const char*)a.p;
    if (d >= bytes(a) || -d >= bytes(b)) return false;
    // Parts of one buffer: with equal strides an element is common where  d + v - u = i * ld + j * bs,  u and v in the rows' widths and
    // i, j differences of frames and sequences; for other strides crossing ranges count as shared.
    if (a.es != b.es || d % a.es || (a.T > 1 && b.T > 1 && a.ld != b.ld) || (a.B > 1 && b.B > 1 && a.bs != b.bs)) return true;
    int64_t ld = a.T > 1 ? a.ld : b.T > 1 ? b.ld : 1, bs = a.B > 1 ? a.bs : b.B > 1 ? b.bs : 1;
    if (ld <= 0 || bs <= 0) return true;
    if (bs < ld) {          // frames outermost: j counts along the longer stride, so that few j are possible
        std::swap(ld, bs);
        std::swap(a.T, a.B);
        std::swap(b.T, b.B);
    }
    a.ld = b.ld = ld;
    const int64_t e = d / a.es;
    auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
    const int64_t lo = std::max(1 - b.B, -floor_div(span(a) - e, bs)), hi = std::min(a.B - 1, floor_div(e + span(b), bs));
    if (hi - lo > 64) return true;                                  // (sequences that lie across one another)
    for (int64_t j = lo; j <= hi; ++j) {
        const int64_t r = e - j * bs;                               // i * ld in (r - a.width, r + b.width)
        if (std::max(1 - b.T, floor_div(r - a.width, ld) + 1) <= std::min(a.T - 1, floor_div(r + b.width - 1, ld))) return true;
    }
    return false;
}

static inline StesRows stes_flat(const void* p, int es, int64_t n) { return StesRows{p, es, n, n, 1, 1, n}; }

// Whether anything that a call writes shares memory with something else that it writes or reads, but for the pair (fine_out, fine_in).
template <int N, int M>
static inline bool stes_any_shared(const StesRows (&outs)[N], const StesRows (&ins)[M], int fine_out = -1, int fine_in = -1) {
    for (int i = 0; i < N; ++i) {
        for (int j = 0; j < M; ++j)
            if (!(i == fine_out && j == fine_in) && stes_share(outs[i], ins[j])) return true;
        for (int j = 0; j < i; ++j)
            if (stes_share(outs[i], outs[j])) return true;
    }
    return false;
}
