// Checks of arguments that the host translation units share.
#pragma once
#include "../../include/alpha_conv_b200.h"
#include "host_common.h"

#include <initializer_list>
#include <stdint.h>

namespace alpha {

inline size_t type_bytes(int dtype) { return dtype == ALPHA_F32 ? 4 : 2; }
inline bool known_type(int dtype) { return dtype == ALPHA_F32 || dtype == ALPHA_BF16 || dtype == ALPHA_F16; }

struct Span { const void* ptr; size_t bytes; };
inline bool overlap(const Span& a, const Span& b)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.ptr), y = reinterpret_cast<uintptr_t>(b.ptr);
    return a.ptr && b.ptr && x < y + b.bytes && y < x + a.bytes;
}
// What a call writes must overlap neither what it reads nor what else it writes.
inline int check_overlaps(const char* what, std::initializer_list<Span> in, std::initializer_list<Span> out)
{
    for (const Span* o = out.begin(); o != out.end(); ++o) {
        for (const Span& i : in)
            if (overlap(*o, i)) return fail(ALPHA_E_ARG, "%s: an output overlaps an input", what);
        for (const Span* q = out.begin(); q != o; ++q)
            if (overlap(*o, *q)) return fail(ALPHA_E_ARG, "%s: two outputs overlap", what);
    }
    return ALPHA_OK;
}
// The same, and every tensor starts on a 16-byte boundary.
inline int check_spans(const char* what, std::initializer_list<Span> in, std::initializer_list<Span> out)
{
    const int rc = check_overlaps(what, in, out);
    if (rc) return rc;
    for (auto list : {in, out})
        for (const Span& s : list)
            if (reinterpret_cast<uintptr_t>(s.ptr) & 15) return fail(ALPHA_E_ARG, "%s: tensor pointers must be 16-byte aligned", what);
    return ALPHA_OK;
}

inline int launched(const char* what)
{
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? ALPHA_OK : fail(ALPHA_E_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
}

}  // namespace alpha
