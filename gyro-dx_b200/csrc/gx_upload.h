// gx_upload.h — a device buffer that is filled from host memory and takes the place of the one before, plain C++
// over a few device calls so that tests/upload_emu.cpp runs it with a device that fails.
#pragma once
#include <stdint.h>

#include "../../include/gyro_moe.h"

namespace gx {

struct HostPiece {
    const void *src;  // nullptr: left as it is
    uint64_t offset, bytes;
};

// held: the buffer in use, or nullptr. On GX_OK it is a new one of the given size that holds the pieces (or, of size
// 0, none), and the old one is gone; on any error it is the old one as it was. dev: alloc(bytes, &p),
// copy(dst, src, bytes) and wait() answer a gx_result, copies are enqueued where the work that reads the buffer is,
// wait() ends when all of it is complete, and release(p) frees.
template <class Dev>
gx_result replace_buffer(Dev &dev, void *&held, uint64_t bytes, const HostPiece *pieces, int n) {
    void *fresh = nullptr;
    gx_result r = bytes ? dev.alloc(bytes, &fresh) : (gx_result)GX_OK;
    if (r != GX_OK) return r;
    for (int i = 0; i < n && r == GX_OK; ++i)
        if (pieces[i].src) r = dev.copy(static_cast<uint8_t *>(fresh) + pieces[i].offset, pieces[i].src, pieces[i].bytes);
    // the copies have arrived, and nothing enqueued before still reads the old buffer
    const gx_result w = dev.wait();
    if (r == GX_OK) r = w;
    if (r != GX_OK) {
        if (fresh && w != GX_E_TIMEOUT) dev.release(fresh);  // after a timeout a copy may still write it
        return r;
    }
    if (held) dev.release(held);
    held = fresh;
    return GX_OK;
}

}  // namespace gx
