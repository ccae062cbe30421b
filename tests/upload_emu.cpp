// gx::replace_buffer (csrc/gx_upload.h) on a device that a test makes fail: copies arrive only in wait().
#include <cstring>
#include <map>
#include <vector>

#include "../gyro-dx_b200/csrc/gx_upload.h"

namespace {
struct Device {
    int fail_alloc = 0, fail_copy = -1;
    gx_result answer = GX_OK;  // of wait()
    int copies = 0, released_in_use = 0;
    std::map<uint8_t *, std::vector<uint8_t>> live;
    struct Pending {
        uint8_t *dst;
        std::vector<uint8_t> data;
    };
    std::vector<Pending> pending;
    gx_result alloc(uint64_t bytes, void **p) {
        if (fail_alloc) return GX_E_OUTOFMEMORY;
        std::vector<uint8_t> v(bytes, 0xee);
        uint8_t *at = v.data();
        live.emplace(at, std::move(v));
        *p = at;
        return GX_OK;
    }
    gx_result copy(void *dst, const void *src, uint64_t bytes) {
        if (copies++ == fail_copy) return GX_E_DEVICE;
        const uint8_t *s = static_cast<const uint8_t *>(src);
        pending.push_back({static_cast<uint8_t *>(dst), {s, s + bytes}});
        return GX_OK;
    }
    gx_result wait() {
        if (answer == GX_E_TIMEOUT) return answer;
        for (auto &p : pending) std::memcpy(p.dst, p.data.data(), p.data.size());
        pending.clear();
        return answer;
    }
    void release(void *p) {
        auto it = live.find(static_cast<uint8_t *>(p));
        for (auto &q : pending)
            if (q.dst >= it->first && q.dst < it->first + it->second.size()) ++released_in_use;
        if (!released_in_use) live.erase(it);
    }
};
}  // namespace

// Fills a buffer with the bytes 1, then replaces it by the bytes 2 in three pieces, the second of them absent. out:
// the 12 bytes in use afterwards, how many buffers live, and whether one was freed under a copy.
extern "C" int replace_twice(int fail_alloc, int fail_copy, int answer, int remove, uint8_t *out, int *live, int *in_use) {
    Device dev;
    void *held = nullptr;
    const std::vector<uint8_t> one(12, 1), two(12, 2);
    const gx::HostPiece a[1] = {{one.data(), 0, 12}};
    if (gx::replace_buffer(dev, held, 12, a, 1) != GX_OK) return 1;
    dev.fail_alloc = fail_alloc;
    dev.copies = 0;
    dev.fail_copy = fail_copy;
    dev.answer = (gx_result)answer;
    const gx::HostPiece b[3] = {{two.data(), 0, 4}, {nullptr, 4, 4}, {two.data(), 8, 4}};
    const gx_result r = remove ? gx::replace_buffer(dev, held, 0, nullptr, 0) : gx::replace_buffer(dev, held, 12, b, 3);
    if (held) std::memcpy(out, held, 12);
    *live = (int)dev.live.size();
    *in_use = dev.released_in_use;
    return r;
}
