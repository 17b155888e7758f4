// peer_rules.hpp -- decisions of the peer transport (peer.hpp) that need no device, apart from it so that they are tested without one:
// when a window may be used again.
#pragma once
#include <cstddef>
#include <cstdint>
#include <mutex>
#include <vector>

namespace nmfx {

// Windows are never freed: memory that was allocated uncached and read by a kernel must not go back to the runtime (allocations that got it
// afterwards have held wrong values).  They are used again, but only once every rank that may have mapped one has said that it will touch it no
// more: a peer that is still solving (it may not have noticed yet that this rank is gone) stores slots, flags and the abort word into it, and the
// next communicator, whose sequence numbers start over, would take them for its own.  A rank says so by storing 1 into its word `ended[rank]` of
// every window it mapped, behind its last exchange (peer.hpp).  A window that some rank never let go of (its process died, or could not map) is
// never used again.  So a process that makes communicators of ever larger windows keeps all of them, and one that repeats a size keeps one a rank.
struct WindowPool {
    struct Kept { int dev; unsigned flags; size_t bytes; unsigned char *p; uint32_t held; };   // held: bit q: rank q may still touch it
    std::mutex m;
    std::vector<Kept> kept;
    // The smallest kept window that serves and that nobody holds, or NULL.  ended(p) gives the ranks that have let go of window p, a bit each.
    template <typename Ended> unsigned char *take(int dev, unsigned flags, size_t &bytes, Ended &&ended) {
        std::lock_guard<std::mutex> lock(m);
        size_t best = kept.size();
        for (size_t i = 0; i < kept.size(); ++i) {
            Kept &k = kept[i];
            if (k.dev != dev || k.flags != flags || k.bytes < bytes || (best < kept.size() && kept[best].bytes <= k.bytes)) continue;
            if (k.held) k.held &= ~ended(k.p);
            if (!k.held) best = i;
        }
        if (best == kept.size()) return nullptr;
        unsigned char *p = kept[best].p;
        bytes = kept[best].bytes;
        kept.erase(kept.begin() + (ptrdiff_t)best);
        return p;
    }
    void give(int dev, unsigned flags, size_t bytes, unsigned char *p, uint32_t held) {
        std::lock_guard<std::mutex> lock(m);
        kept.push_back(Kept{dev, flags, bytes, p, held});
    }
};

}  // namespace nmfx
