// Pieces of memory that a call writes and reads, and what it may not be handed.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <initializer_list>

#include "bank.h"

namespace kiln {

struct Piece {
    const void *at;
    size_t bytes;
};
// does anything written share memory with anything read, or with something else written?  (Nothing at null, or of no bytes, does.)
inline bool any_meet(std::initializer_list<Piece> written, std::initializer_list<Piece> read) {
    auto share = [](const Piece &a, const Piece &b) { return a.at && b.at && a.bytes && b.bytes && meet(a.at, a.bytes, b.at, b.bytes); };
    for (const Piece *w = written.begin(); w != written.end(); ++w) {
        for (const Piece *v = w + 1; v != written.end(); ++v)
            if (share(*w, *v)) return true;
        for (const Piece &r : read)
            if (share(*w, r)) return true;
    }
    return false;
}
// may one launch have so many blocks?  (Its work-items are counted in 32 bits.)
inline bool launchable(int64_t blocks, int threads) { return blocks * threads <= (int64_t)UINT32_MAX; }
// all there and on `bytes`?
inline bool all_on(size_t bytes, std::initializer_list<const void *> pointers) {
    for (const void *p : pointers)
        if (!p || reinterpret_cast<uintptr_t>(p) % bytes != 0) return false;
    return true;
}

}  // namespace kiln
