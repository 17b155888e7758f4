// peer_rules.hpp -- decisions of the peer transport (peer.hpp) that need no device, apart from it so that they are tested without one:
// when a window may be used again, and which layouts of ranks over devices and processes are refused.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cstdlib>
#include <mutex>
#include <string>
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

// A number for a device, the same for two ranks only where they certainly use the same one: partitions of a card are devices of their own with one
// PCI address, so a process's number of the device and what it sees of them count too.
inline uint64_t device_place(const char *pci, int number, const char *visible, const char *visible_to_rocr) {
    uint64_t h = 0xcbf29ce484222325ull;
    auto add = [&](const char *s) {
        for (; s && *s; ++s) h = (h ^ (unsigned char)*s) * 0x100000001b3ull;
        h = (h ^ 0x1ffu) * 0x100000001b3ull;          // (no character)
    };
    add(pci);
    add(std::to_string(number).c_str());
    add(visible);
    add(visible_to_rocr);
    return h;
}
// Where a rank is.  device: as above; queues: hardware queues that the rank's process has on a device.
struct PeerPlace {
    int32_t pid, queues;
    uint64_t device, window;
};
// HIP spreads a process's streams over GPU_MAX_HW_QUEUES hardware queues, 4 unless it says otherwise.
inline int hw_queues(const char *setting) {
    const int n = setting ? std::atoi(setting) : 0;
    return n > 0 ? n : 4;
}
// Ranks that share a device wait for each other with kernels that spin, so what a wait is for must get to run beside it.
//  * In one process a signal that sits in one hardware queue behind another rank's wait never runs (the wait ends by its time-out).  A rank has
//    up to three streams and the process its default one: with a queue for each nothing sits behind anything.  Four ranks: with 4 queues they
//    time out, with 8 now and then, with 24 never.  Two ranks' exchanging streams have queues of their own with the default 4 as well.
//  * Of processes on one device two run; with four of them the GPU has stood still, and the cause is not known.
// Every rank has the same places and comes to the same answer.  NULL: the layout is fine.
inline const char *peer_layout_refusal(const PeerPlace *at, int n) {
    for (int i = 0; i < n; ++i) {
        int processes = 0, ranks = 0;
        for (int q = 0; q < n; ++q) {
            if (at[q].device != at[i].device) continue;
            bool new_process = true, new_rank = at[q].pid == at[i].pid;      // (the timing stand-in names one window several times)
            for (int r = 0; r < q; ++r) {
                new_process = new_process && !(at[r].device == at[q].device && at[r].pid == at[q].pid);
                new_rank = new_rank && !(at[r].device == at[q].device && at[r].pid == at[q].pid && at[r].window == at[q].window);
            }
            processes += new_process;
            ranks += new_rank;
        }
        if (processes > 2) return "peer attach: more than two processes on one device (their kernels wait for each other and may never run side by side): use one device per process";
        if (ranks > 1 && at[i].queues < (ranks == 2 ? 4 : 3 * ranks + 1))
            return "peer attach: several ranks of one process on one device need a hardware queue for each of their streams: set GPU_MAX_HW_QUEUES to 3 a rank and one more before the process uses the GPU, or use the in-process group";
    }
    return nullptr;
}

}  // namespace nmfx
