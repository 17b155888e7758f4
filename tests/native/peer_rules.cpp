// csrc/peer_rules.hpp behind plain C functions, for tests/test_peer_rules.py (no device is used: a window is a number here)
#include <map>

#include "../../nmf.jl_amd/csrc/peer_rules.hpp"

static std::map<unsigned char *, uint32_t> ended;

extern "C" {
void *pool_new() { ended.clear(); return new nmfx::WindowPool; }
void pool_delete(void *pool) { delete static_cast<nmfx::WindowPool *>(pool); }
void pool_give(void *pool, int dev, unsigned flags, uint64_t bytes, uint64_t window, unsigned held) {
    static_cast<nmfx::WindowPool *>(pool)->give(dev, flags, (size_t)bytes, reinterpret_cast<unsigned char *>(window), held);
}
// rank q stores its word into a window
void window_end(uint64_t window, int q) { ended[reinterpret_cast<unsigned char *>(window)] |= 1u << q; }
// 0: none; *bytes: what is asked for, and what it has
uint64_t pool_take(void *pool, int dev, unsigned flags, uint64_t *bytes) {
    size_t b = (size_t)*bytes;
    unsigned char *p = static_cast<nmfx::WindowPool *>(pool)->take(dev, flags, b, [](const unsigned char *w) { return ended[const_cast<unsigned char *>(w)]; });
    *bytes = b;
    return reinterpret_cast<uint64_t>(p);
}
uint64_t place_of(const char *pci, int number, const char *visible, const char *visible_to_rocr) { return nmfx::device_place(pci, number, visible, visible_to_rocr); }
int queues_of(const char *setting) { return nmfx::hw_queues(setting); }
// ranks as pid, queues, device, window
const char *layout_refusal(const uint64_t *ranks, int n) {
    std::vector<nmfx::PeerPlace> at;
    for (int i = 0; i < n; ++i) at.push_back(nmfx::PeerPlace{(int32_t)ranks[4 * i], (int32_t)ranks[4 * i + 1], ranks[4 * i + 2], ranks[4 * i + 3]});
    return nmfx::peer_layout_refusal(at.data(), n);
}
}
