// What the tiled block-scaled E4M3 products (fp8_gemm.hip, fp8_glu.hip) share:
// direct-to-LDS loads and their waits, and the rows of a tile.
#pragma once

#include "fp8.hpp"

namespace kmi {

constexpr uint32_t G_NONE = 0x80000000u;     // past every view: reads 0
constexpr int G_CHUNK = 64;                  // blocks whose scales are held at a time

template <int N_>
__device__ __forceinline__ void g_wait() {
    static_assert(N_ >= 0 && N_ < 64, "vmcnt");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N_) : "memory");
}

// 16 bytes per lane from the view's offset into LDS at byte dst + 16 lane.  In asm,
// as the compiler would wait for the load before any later read of LDS; the kernel
// waits for it itself (g_wait), and the compiler's own counts, which miss these
// loads, only wait for more.
__device__ __forceinline__ void g_dma16(__amdgpu_buffer_rsrc_t r, uint32_t dst, uint32_t voff, uint32_t soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 ::"s"(dst), "v"(voff), "s"(r), "s"(soff) : "memory", "m0");
}
// the byte address of shared memory p (taken once: a generic pointer's conversion
// tests for null every time)
__device__ __forceinline__ uint32_t g_lds(const void* p) {
    return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p);
}

// A tile: (expert, first row, rows) of the list, or rows [a.tm z, ..) of expert 0.
struct GTile {
    int64_t expert, start;
    int count;
};
__device__ __forceinline__ GTile g_tile(const F8Args& a, int tile) {
    if (!a.tiles) {
        const int64_t start = (int64_t)tile * a.tm;
        return {0, start, (int)(a.rows - start < a.tm ? a.rows - start : a.tm)};
    }
    // (through the scalar cache: one load for the wave)
    typedef const __attribute__((address_space(4))) int32_t* sptr;
    const sptr t = (sptr)(uintptr_t)(a.tiles + 3 * (int64_t)tile);
    return {t[0], t[1], t[2]};
}

// x rows of rows m0, m0 + by, .. of a tile, or -1: every load of a kind before the
// first is waited for (a workgroup's start is a chain of such latencies)
template <int N>
__device__ __forceinline__ void g_xrows(const F8Args& a, const GTile& t, int m0, int by, int64_t (&row)[N]) {
    if (!a.tiles || a.in_order) {
#pragma unroll
        for (int j = 0; j < N; j++) row[j] = m0 + by * j < t.count ? t.start + m0 + by * j : -1;
        return;
    }
    int p[N], in[N], b[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
        const int m = m0 + by * j;
        p[j] = a.sorted[t.start + (m < t.count ? m : t.count - 1)];
        in[j] = 0;
    }
    if (a.Mper != 1) {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int rid = p[j];
            p[j] = rid / (int)a.Mper;
            in[j] = rid - p[j] * (int)a.Mper;
        }
    }
    if (a.lhs) {
#pragma unroll
        for (int j = 0; j < N; j++) b[j] = a.lhs[p[j]];
    } else {
        // p / lhs_div: half a step from every border, so exact in float64
#pragma unroll
        for (int j = 0; j < N; j++) b[j] = (int)(((double)p[j] + 0.5) * a.lhs_inv);
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
        const int64_t r = (int64_t)b[j] * a.Mper + in[j];
        row[j] = m0 + by * j < t.count && b[j] >= 0 && r < a.xrows ? r : -1;
    }
}

// The scale bytes of a tile's TM rows, G_CHUNK blocks from t0, by direct-to-LDS
// loads into sc[G_CHUNK / 16][TM][16]: g_scale_loads per wave.
template <int TM, int WAVES>
constexpr int g_scale_loads = (G_CHUNK / 16 * TM / 64 + WAVES - 1) / WAVES;
template <int TM, int WAVES>
__device__ __forceinline__ void g_scales(const F8Args& a, const GTile& tile, uint32_t sc, int t0, int KB, int wave,
                                         int lane) {
    constexpr int N = g_scale_loads<TM, WAVES>, G = TM / 64;
    static_assert(N * WAVES == G_CHUNK / 16 * G, "whole loads per wave");
    const int64_t x0 = a.tiles ? 0 : tile.start;
    const __amdgpu_buffer_rsrc_t r = make_rsrc(a.xs + x0 * a.xs_ld, (a.xrows - x0) * a.xs_ld);
    static_assert(G == 1 || WAVES % G == 0, "a wave's loads are of the same rows");
    int64_t row[1];
    g_xrows(a, tile, 64 * (wave % G) + lane, 0, row);
    uint32_t off[N];
#pragma unroll
    for (int i = 0; i < N; i++) {                // 16 blocks' piece u / G, 64 rows u % G
        const int t = t0 + 16 * ((wave + WAVES * i) / G);
        off[i] = row[0] >= 0 && t < KB ? (uint32_t)((row[0] - x0) * a.xs_ld) + t : G_NONE;
    }
#pragma unroll
    for (int i = 0; i < N; i++) g_dma16(r, sc + (wave + WAVES * i) * 1024, off[i], 0);
}
__device__ __forceinline__ uint32_t g_scale(const unsigned char* sc, int TM, int row, int t) {
    return sc[(t % G_CHUNK / 16 * TM + row) * 16 + t % 16];
}

// Grouped tiles: workgroup -> (tile, column block).  Workgroups go to the 8 XCDs
// in turn.  A unit is 4 neighbouring tiles (often one expert's) x `cols` column
// blocks: it stays on one XCD, whose L2 then serves its weights to the other tiles
// and its rows to the other columns; the next unit goes to the next XCD.  Units of
// up to 4, all alike (a last one of 2 of 6 columns left half the XCDs a third less:
// 302 us for 276): with all columns in one, few tiles fill few XCDs (512 rows of 8 experts
// [4096, 4096]: 92.6 us, 53.8 so); with 1, many tiles' rows go through every L2
// (32768 rows of 128 experts [1536, 4096]: 500 us, 474 so).
struct GPlace {
    int units, cols;            // units to a group of 4 tiles, column blocks to a unit
};
__device__ __forceinline__ void g_place(int id, GPlace p, int& tile, int& nb) {
    const int kk = id >> 3, v = kk / (4 * p.cols), u = v * 8 + (id & 7), in = kk - 4 * p.cols * v;
    tile = u / p.units * 4 + in % 4;
    nb = u % p.units * p.cols + in / 4;
}
inline GPlace g_place_of(int64_t nblocks) {
    const int64_t cols = nblocks % 4 == 0 ? 4 : nblocks % 3 == 0 ? 3 : nblocks % 2 == 0 ? 2 : 1;
    return {(int)ceil_div(nblocks, cols), (int)cols};
}
inline int64_t g_place_grid(int64_t tiles, GPlace p) {
    return ceil_div(ceil_div(tiles, 4) * p.units, 8) * 32 * p.cols;
}

}  // namespace kmi
