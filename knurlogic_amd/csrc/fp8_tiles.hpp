// What the tiled block-scaled E4M3 products (fp8_gemm.hip, fp8_glu.hip) share:
// direct-to-LDS loads and their waits, and the rows of a tile.
#pragma once

#include "fp8.hpp"

namespace kmi {

#define KMI_F8_LDS(p) ((__attribute__((address_space(3))) unsigned char*)(p))

constexpr uint32_t G_NONE = 0x80000000u;     // past every view: reads 0
constexpr int G_CHUNK = 64;                  // blocks whose scales are held at a time

template <int N_>
__device__ __forceinline__ void g_wait() {
    static_assert(N_ >= 0 && N_ < 64, "vmcnt");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N_) : "memory");
}

// 16 bytes per lane from the view's offset into LDS at dst + 16 lane.  In asm, as
// the compiler would wait for the load before any later read of LDS; the kernel
// waits for it itself (g_wait), and the compiler's own counts, which miss these
// loads, only wait for more.
__device__ __forceinline__ void g_dma16(__amdgpu_buffer_rsrc_t r, unsigned char* dst, uint32_t voff, uint32_t soff) {
    const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)KMI_F8_LDS(dst));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 ::"s"(at), "v"(voff), "s"(r), "s"(soff) : "memory", "m0");
}

// x row of row m of a tile of `count` rows from `start`, or -1
__device__ __forceinline__ int64_t g_xrow(const F8Args& a, int64_t start, int count, int m) {
    if (m >= count) return -1;
    if (!a.tiles) return start + m;
    const int rid = a.sorted[start + m];
    const int p = rid / (int)a.Mper;
    const int64_t b = a.lhs ? a.lhs[p] : p / (int)a.lhs_div;
    const int64_t r = b * a.Mper + rid % (int)a.Mper;
    return b >= 0 && r < a.xrows ? r : -1;
}

// Grouped tiles: workgroup -> (tile, column block).  Workgroups go to the 8 XCDs
// in turn; 2 neighbouring tiles (often one expert's) of every column block stay on
// one XCD, whose L2 then serves the second, the next 2 go to the next (tiles at
// the list's end are empty: they must not all fall to one).
__device__ __forceinline__ void g_place(int id, int nblocks, int& tile, int& nb) {
    const int xcd = id & 7, kk = id >> 3;
    tile = ((kk / (2 * nblocks)) * 8 + xcd) * 2 + kk % 2;
    nb = kk / 2 % nblocks;
}
inline int64_t g_place_grid(int64_t tiles, int64_t nblocks) { return ceil_div(tiles, 16) * 16 * nblocks; }

}  // namespace kmi
