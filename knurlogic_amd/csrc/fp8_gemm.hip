// Block-scaled E4M3 products of many rows: tiles of 256 weight rows (gate|up: 128
// gate and 128 up rows) x 64 to 256 activation rows.
//
// The rows of x are quantized by a pass before (f8_rows).  4 or 8 waves take 64
// weight rows x MB 16-row blocks of activations each.  Both operands arrive by
// direct-to-LDS loads, S blocks of 128 inputs in a ring: 8 lanes take the 128
// bytes of a row (straight into the operand, a lane per row, the address units
// handled a lane at a time: 4900 of 6300 cycles per block), their 16-byte pieces
// permuted by the row, so that 8 rows' reads fall on distinct banks.  The
// barrier of a block stands before its last products, where all of its LDS reads
// are done: those products run while the next block's first fragments are read.
// D holds activation rows along its columns, so a lane has one row's scale per
// 16 x 16 tile.
#include "fp8.hpp"

namespace kmi {

namespace {

#define KMI_F8_LDS(p) ((__attribute__((address_space(3))) unsigned char*)(p))

constexpr uint32_t G_NONE = 0x80000000u;     // past every view: reads 0
constexpr int G_CHUNK = 64;                  // blocks whose scales are held at a time

// how weights and x meet: E4M3 operands with both scales applied to each
// block's sums in float32 (weights' scales in float32), or by the instruction
// (E8M0); or float16 operands (gate|up, whose results are rounded to E4M3 again)
enum Kind { F32S, E8S, HALF };

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

// NW x WM waves: 64 weight rows x MB 16-row blocks of activations each
template <int NW, int WM, int MB, int S>
struct Shape {
    static constexpr int TN = 64 * NW, TM = 16 * MB * WM, WAVES = NW * WM;
    static constexpr int WTILE = TN * F8_BLOCK, STAGE = WTILE + TM * F8_BLOCK;   // a block's bytes in LDS
    static constexpr int XL = TM / 8 / WAVES, WL = TN / 8 / WAVES;               // loads per wave and block
    static constexpr int LDS = S * STAGE + G_CHUNK * TM;
    static_assert(XL * 8 * WAVES == TM && WL * 8 * WAVES == TN, "whole loads per wave");
};

template <Kind KIND, int NW, int WM, int MB, int S, bool GLU>
__global__ __launch_bounds__(64 * NW * WM, 2) void f8_gemm(F8Args a, int nblocks, int tiles) {
    typedef Shape<NW, WM, MB, S> Z;
    static_assert(!GLU || NW == 4, "gate|up: 128 columns per workgroup");
    constexpr int RB = 4, TN = Z::TN, TM = Z::TM, XL = Z::XL, WL = Z::WL, WAVES = Z::WAVES, WTILE = Z::WTILE;
    constexpr int COLS = GLU ? TN / 2 : TN;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int rid_s[TM];
    unsigned char* const sc = smem + S * Z::STAGE;            // [G_CHUNK][WM][16][MB] scale bytes
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave % NW, wm = wave / NW;
    const int l16 = lane & 15, c = lane >> 4;
    // workgroup -> (tile, column block).  Workgroups go to the 8 XCDs in turn, and
    // an XCD's neighbours should share weights and x in its L2.  Dense: each XCD
    // takes an eighth of the (tile, column block) pairs, in strips of 8 tiles.
    // Grouped: 2 neighbouring tiles (often one expert's) of every column block on
    // one XCD, the next 2 on the next (tiles at the list's end are empty: they
    // must not all fall to one)
    const int xcd = (int)blockIdx.x & 7, kk = (int)blockIdx.x >> 3;
    int tile, nb;
    if (a.tiles) {
        tile = ((kk / (2 * nblocks)) * 8 + xcd) * 2 + kk % 2;
        nb = kk / 2 % nblocks;
        if (tile >= tiles) return;
    } else {
        const int idx = xcd * ((int)gridDim.x >> 3) + kk, strip = idx / (8 * nblocks), in = idx - strip * 8 * nblocks;
        if (idx >= tiles * nblocks) return;
        const int height = tiles - 8 * strip < 8 ? tiles - 8 * strip : 8;
        tile = 8 * strip + in % height;
        nb = in / height;
    }
    int64_t expert = 0, start = (int64_t)tile * a.tm;
    int count = (int)(a.rows - start < a.tm ? a.rows - start : a.tm);
    if (a.tiles) {
        const int32_t* t = a.tiles + 3 * (int64_t)tile;
        expert = t[0]; start = t[1]; count = t[2];
    }
    if (count <= 0) return;

    const int K = (int)a.K, KB = (K + F8_BLOCK - 1) / F8_BLOCK;
    const int64_t x0 = a.tiles ? 0 : start;                   // the x view's first row
    auto xrow = [&](int m) -> int64_t {                       // x row of tile row m, or -1
        if (m >= count) return -1;
        if (!a.tiles) return start + m;
        const int rid = a.sorted[start + m];
        const int p = rid / (int)a.Mper;
        const int64_t b = a.lhs ? a.lhs[p] : p / (int)a.lhs_div;
        const int64_t r = b * a.Mper + rid % (int)a.Mper;
        return b >= 0 && r < a.xrows ? r : -1;
    };
    // direct-to-LDS loads: 8 lanes per row, the lane's piece permuted by the row
    const int piece = (lane & 7) ^ (lane >> 3);               // (row % 8 == lane / 8)
    const __amdgpu_buffer_rsrc_t rx = make_rsrc((const unsigned char*)a.x + x0 * a.xld, (a.xrows - x0) * a.xld);
    uint32_t xoff[XL], woff[WL];
#pragma unroll
    for (int j = 0; j < XL; j++) {
        const int64_t r = xrow(8 * (wave + WAVES * j) + (lane >> 3));
        xoff[j] = r < 0 ? G_NONE : (uint32_t)((r - x0) * a.xld) + 16u * piece;
    }
    // weight rows of the tile: row 64 v + 16 i + l of wave column v's fragment i
    // (gate|up: fragments 0, 1 the gate rows 32 v .., 2, 3 the up rows)
    const int64_t n0 = (int64_t)nb * COLS;
    const int64_t left = a.N - n0 < COLS ? a.N - n0 : COLS;
    const __amdgpu_buffer_rsrc_t rw = make_rsrc(a.w + (expert * a.wrows + n0) * a.K, left * a.K);
    const __amdgpu_buffer_rsrc_t ru = make_rsrc(a.w + (expert * a.wrows + n0 + (GLU ? a.N : 0)) * a.K, left * a.K);
#pragma unroll
    for (int j = 0; j < WL; j++) {
        const int m = 8 * (wave + WAVES * j) + (lane >> 3);
        const int r = GLU ? (m >> 6) * 32 + (m & 31) : m;     // (bit 5 of m: up)
        woff[j] = r < left ? (uint32_t)r * (uint32_t)K + 16u * piece : G_NONE;
    }
    auto issue = [&](int t) {                                 // block t (past the last: zeros)
        unsigned char* dst = smem + (t % S) * Z::STAGE;
        const bool in = t * F8_BLOCK + 16 * piece < K;        // inputs past the last: zeros
#pragma unroll
        for (int j = 0; j < WL; j++) {
            const int m = 8 * (wave + WAVES * j);
            g_dma16(GLU && (m & 32) ? ru : rw, dst + m * F8_BLOCK, in ? woff[j] : G_NONE, (uint32_t)t * F8_BLOCK);
        }
#pragma unroll
        for (int j = 0; j < XL; j++)
            g_dma16(rx, dst + WTILE + (wave + WAVES * j) * 1024, t < KB ? xoff[j] : G_NONE, (uint32_t)t * F8_BLOCK);
    };
#pragma unroll
    for (int t = 0; t < S; t++) issue(t);
    // the weights' scales of the wave's rows, 64 blocks, one per lane (gate|up:
    // gate, up), and the scale bytes of x's rows
    const int64_t SB = (a.wrows + F8_BLOCK - 1) / F8_BLOCK;
    const int64_t nw = n0 + (GLU ? 0 : 64 * wn);
    const int64_t sbase = (expert * SB + (nw < a.N ? nw : n0) / F8_BLOCK) * KB;
    uint32_t swl[GLU ? 2 : 1];
    auto load_scales = [&](int t) {
        const int k = t + lane < KB ? t + lane : KB - 1;
#pragma unroll
        for (int g = 0; g < (GLU ? 2 : 1); g++) {
            const int64_t i = sbase + (g ? a.N / F8_BLOCK * KB : 0) + k;
            if (KIND == E8S) swl[g] = ((const unsigned char*)a.s)[i];
            else if (a.e8) swl[g] = __float_as_uint(e8m0_to_f32(((const unsigned char*)a.s)[i]));
            else swl[g] = ((const uint32_t*)a.s)[i];
        }
#pragma unroll
        for (int g = 0; g < (GLU ? 2 : 1); g++) asm volatile("" : "+v"(swl[g]));     // waited for here, not in the loop
        for (int m = tid & (TM - 1), q = tid / TM; q < G_CHUNK / 4 && t + 4 * q < KB; q += 64 * WAVES / TM) {
            const int64_t r = xrow(m);
            const uint32_t v = r < 0 ? 0x7f7f7f7fu : *(const uint32_t*)(a.xs + r * a.xs_ld + t + 4 * q);
            const int w = m / (16 * MB), j = m / 16 % MB;
#pragma unroll
            for (int b = 0; b < 4; b++)
                sc[(((4 * q + b) * WM + w) * 16 + (m & 15)) * MB + j] = (unsigned char)(v >> (8 * b));
        }
    };
    load_scales(0);
    if (tid < TM) rid_s[tid] = tid >= count ? -1 : a.tiles ? a.sorted[start + tid] : (int)(start + tid);

    // fragment reads: weight row 64 wn + 16 i + l16, pieces c and c + 4; x row
    // 16 (MB wm + j) + l16, the same
    uint32_t xo[2], wo[2];
#pragma unroll
    for (int q = 0; q < 2; q++) {
        wo[q] = (uint32_t)(64 * wn + l16) * F8_BLOCK + 16u * ((c + 4 * q) ^ (l16 & 7));
        xo[q] = WTILE + (uint32_t)(16 * MB * wm + l16) * F8_BLOCK + 16u * ((c + 4 * q) ^ (l16 & 7));
    }
    i32x8 w[RB], b[2];
    auto read_w = [&](const unsigned char* st, int i) {
        w[i] = f8_operand(*(const u32x4*)(st + i * 2048 + wo[0]), *(const u32x4*)(st + i * 2048 + wo[1]));
    };
    auto read_b = [&](const unsigned char* st, int j) {
        b[j & 1] = f8_operand(*(const u32x4*)(st + j * 2048 + xo[0]), *(const u32x4*)(st + j * 2048 + xo[1]));
    };
    f32x4 acc[RB][MB];
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int j = 0; j < MB; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    g_wait<(S - 1) * (XL + WL)>();
    lds_barrier();
#pragma unroll
    for (int i = 0; i < RB; i++) read_w(smem, i);
    read_b(smem, 0);
    static_assert(MB % 2 == 0, "x fragments alternate");
    for (int t0 = 0; t0 < KB; t0 += G_CHUNK) {
    if (t0) {                                    // every wave is past its reads of the last chunk's scales
        load_scales(t0);
        lds_barrier();
    }
    const int t1 = t0 + G_CHUNK < KB ? t0 + G_CHUNK : KB;
    for (int t = t0; t < t1; t++) {              // (no branch inside: the compiler would sink products past it)
        const unsigned char* st = smem + (t % S) * Z::STAGE;
        const unsigned char* nx = smem + ((t + 1) % S) * Z::STAGE;
        uint32_t sx[(MB + 3) / 4];
        const unsigned char* sp = sc + ((t % G_CHUNK * WM + wm) * 16 + l16) * MB;
        if constexpr (MB == 2) {
            sx[0] = *(const uint16_t*)sp;
        } else {
#pragma unroll
            for (int q = 0; q < MB / 4; q++) sx[q] = *(const uint32_t*)(sp + 4 * q);
        }
        uint32_t sw[GLU ? 2 : 1];
#pragma unroll
        for (int g = 0; g < (GLU ? 2 : 1); g++) sw[g] = (uint32_t)__builtin_amdgcn_readlane((int)swl[g], t % G_CHUNK);
        auto row_scale = [&](int j) { return __uint_as_float((sx[j / 4] >> (8 * (j & 3)) & 0xffu) << 23); };
        // after the block's last LDS read: the next block has landed, and this
        // one's place is free
        auto turn = [&]() {
            g_wait<(S - 2) * (XL + WL)>();
            lds_barrier();
            issue(t + S);
        };
        if constexpr (KIND == HALF) {
            typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
            auto halves = [](const i32x8& v, int q) -> f16x8 {       // codes 8 q .. 8 q + 7
                const uint32_t d0 = (uint32_t)v[2 * q], d1 = (uint32_t)v[2 * q + 1];
                const f16x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d0, 1.f, false);
                const f16x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d0, 1.f, true);
                const f16x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d1, 1.f, false);
                const f16x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d1, 1.f, true);
                return f16x8{p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
            };
            f16x8 wh[RB][4];
#pragma unroll
            for (int i = 0; i < RB; i++)
#pragma unroll
                for (int q = 0; q < 4; q++) wh[i][q] = halves(w[i], q);
#pragma unroll
            for (int j = 0; j < MB; j++) {
                if (j + 1 < MB) {
                    read_b(st, j + 1);
                } else {
                    turn();
#pragma unroll
                    for (int i = 0; i < RB; i++) read_w(nx, i);
                }
                const float f = row_scale(j);
                f16x8 bh[4];
#pragma unroll
                for (int q = 0; q < 4; q++) bh[q] = halves(b[j & 1], q);
                f32x4 p[RB];
#pragma unroll
                for (int i = 0; i < RB; i++) p[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int q = 0; q < 4; q++)
#pragma unroll
                    for (int i = 0; i < RB; i++)
                        p[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[i][q], bh[q], p[i], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < RB; i++) {
                    const float g = f * __uint_as_float(sw[GLU && i >= 2 ? 1 : 0]);
#pragma unroll
                    for (int q = 0; q < 4; q++) acc[i][j][q] = __builtin_fmaf(p[i][q], g, acc[i][j][q]);
                }
            }
            read_b(nx, 0);
        } else {
            // product n = 4 j + i; its sums are scaled two products later
            constexpr int NP = RB * MB;
            f32x4 p[3];
            float f[2];
            auto apply = [&](int n) {
                const int i = n % RB, j = n / RB;
#pragma unroll
                for (int q = 0; q < 4; q++) acc[i][j][q] = __builtin_fmaf(p[n % 3][q], f[j & 1], acc[i][j][q]);
            };
#pragma unroll
            for (int n = 0; n < NP; n++) {
                const int i = n % RB, j = n / RB;
                if (i == 0) {
                    if (j + 1 < MB) read_b(st, j + 1);
                    else turn();
                }
                if (n == NP - RB) read_b(nx, 0);
                if constexpr (KIND == E8S) {
                    acc[i][j] = f8_mfma_at(w[i], b[j & 1], acc[i][j], sw[0], sx[j / 4], j & 3);
                } else {
                    if (i == 0) f[j & 1] = row_scale(j) * __uint_as_float(sw[0]);
                    p[n % 3] = f8_mfma(w[i], b[j & 1], f32x4{0.f, 0.f, 0.f, 0.f}, 127u, 127u);
                    if (n >= 2) apply(n - 2);
                }
                if (j == MB - 1) read_w(nx, i);
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (KIND == F32S) {
                apply(NP - 2);
                apply(NP - 1);
            }
        }
    }
    }
    g_wait<0>();                                 // no load still writes LDS below

    if constexpr (GLU) {
        // activations of 128 columns per row through LDS, where 16 lanes quantize
        // a row's group
        lds_barrier();
#pragma unroll
        for (int j = 0; j < MB; j++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                uint32_t o[2];
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    const uint32_t gg = cvt_pk_bf16(acc[i][j][2 * q], acc[i][j][2 * q + 1]);
                    const uint32_t uu = cvt_pk_bf16(acc[i + 2][j][2 * q], acc[i + 2][j][2 * q + 1]);
                    o[q] = cvt_pk_bf16(silu_bf16r(__uint_as_float(gg << 16)) * __uint_as_float(uu << 16),
                                       silu_bf16r(__uint_as_float(gg & 0xffff0000u)) * __uint_as_float(uu & 0xffff0000u));
                }
                *(u32x2*)(smem + (16 * (MB * wm + j) + l16) * 272 + (32 * wn + 16 * i + 4 * c) * 2) = u32x2{o[0], o[1]};
            }
        lds_barrier();
        for (int m = tid >> 4; m < count; m += 4 * WAVES) {
            F8Raw<F8BF16, 8> v;
            v.v[0] = *(const u32x4*)(smem + m * 272 + 16 * l16);
            uint32_t byte = f8_scale_byte(f8_max16(v.amax()));
            const bool nan = byte == 255;        // as f8_rows
            if (nan) byte = 127;
            const float scale = __uint_as_float(byte << 23);
            unsigned char* y = (unsigned char*)a.y + (int64_t)rid_s[m] * a.N + nb * 128 + 8 * l16;
            *(u32x2*)y = nan ? u32x2{0x7f7f7f7fu, 0x7f7f7f7fu} : u32x2{v.codes(0, scale), v.codes(1, scale)};
            if (l16 == 0) a.ys[(int64_t)rid_s[m] * a.ys_ld + nb] = (unsigned char)byte;
        }
    } else {
        uint16_t* y = (uint16_t*)a.y;
        const bool wide = a.N % 4 == 0 && ((uintptr_t)a.y & 7) == 0;
#pragma unroll
        for (int j = 0; j < MB; j++) {
            const int m = 16 * (MB * wm + j) + l16;
            const int rid = rid_s[m];
            if (rid < 0) continue;
            const bool seen = !a.lhs || xrow(m) >= 0;
#pragma unroll
            for (int i = 0; i < RB; i++) {
                const int64_t n = n0 + 64 * wn + 16 * i + 4 * c;
                u32x2 o;
                if (a.half) {
                    o.x = f32_to_f16(acc[i][j][0]) | (uint32_t)f32_to_f16(acc[i][j][1]) << 16;
                    o.y = f32_to_f16(acc[i][j][2]) | (uint32_t)f32_to_f16(acc[i][j][3]) << 16;
                } else {
                    o.x = cvt_pk_bf16(acc[i][j][0], acc[i][j][1]);
                    o.y = cvt_pk_bf16(acc[i][j][2], acc[i][j][3]);
                }
                if (!seen) o = u32x2{0, 0};
                uint16_t* q = y + (int64_t)rid * a.N + n;
                if (wide) {
                    if (n < a.N) *(u32x2*)q = o;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (n + e < a.N) q[e] = (uint16_t)(o[e >> 1] >> (16 * (e & 1)));
                }
            }
        }
    }
}

// x's rows into codes [rows, ld] (tails zero) and scale bytes [rows, sld]: 16
// lanes per row and block.
template <class T>
__global__ __launch_bounds__(256) void f8_rows(const typename T::storage* __restrict__ x, int64_t rows, int K, int KB,
                                               unsigned char* __restrict__ q, int64_t ld,
                                               unsigned char* __restrict__ s, int64_t sld) {
    const int64_t id = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4;
    const int l = threadIdx.x & 15;
    const int64_t r = id / KB;
    const int b = (int)(id % KB), k = b * F8_BLOCK + 8 * l;
    if (r >= rows) return;
    F8Raw<T, 8> v;
    if (k < K) v.load(x + r * K + k);
    else v.zero();
    // a block with an infinity or a NaN: NaN codes, so the scale stays a number
    uint32_t byte = f8_scale_byte(f8_max16(v.amax()));
    const bool nan = byte == 255;
    if (nan) byte = 127;
    const float scale = __uint_as_float(byte << 23);
    *(u32x2*)(q + r * ld + k) = nan ? u32x2{0x7f7f7f7fu, 0x7f7f7f7fu} : u32x2{v.codes(0, scale), v.codes(1, scale)};
    if (l == 0) s[r * sld + b] = (unsigned char)byte;
}

template <Kind KIND, int NW, int WM, int MB, int S, bool GLU>
int go(const F8Args& a, int64_t tiles, hipStream_t st) {
    typedef Shape<NW, WM, MB, S> Z;
    if (a.K > FP8_GEMM_MAX_K || a.xld != fp8_row_bytes(a.K) || a.tm > Z::TM) {
        set_error("fp8: K=%lld in tiles of %d", (long long)a.K, a.tm);
        return EINVAL_ARG;
    }
    const int nblocks = (int)ceil_div(a.N, GLU ? Z::TN / 2 : Z::TN);
    const int64_t wgs = a.tiles ? ceil_div(tiles, 16) * 16 * nblocks : ceil_div(tiles * nblocks, 8) * 8;
    if (wgs >= (1LL << 31)) {
        set_error("fp8: grid of %lld workgroups", (long long)wgs);
        return EINVAL_ARG;
    }
    allow_dynamic_lds_once((const void*)f8_gemm<KIND, NW, WM, MB, S, GLU>);
    f8_gemm<KIND, NW, WM, MB, S, GLU><<<(unsigned)wgs, 64 * Z::WAVES, Z::LDS, st>>>(a, nblocks, (int)tiles);
    KMI_CHECK_LAUNCH("fp8 tiles");
    return OK;
}

template <int NW, int WM, int MB, int S>
int go(const F8Args& a, int64_t tiles, hipStream_t st) {
    return a.e8 ? go<E8S, NW, WM, MB, S, false>(a, tiles, st) : go<F32S, NW, WM, MB, S, false>(a, tiles, st);
}

}  // namespace

int64_t fp8_row_bytes(int64_t K) { return ceil_div(K, F8_BLOCK) * F8_BLOCK; }
int64_t fp8_row_scales(int64_t K) { return ceil_div(ceil_div(K, F8_BLOCK), 4) * 4; }

int launch_fp8_rows(const void* x, int dtype, int64_t rows, int64_t K, unsigned char* q, unsigned char* s,
                    hipStream_t st) {
    const int64_t KB = ceil_div(K, F8_BLOCK), grid = ceil_div(rows * KB, 16);
    if (grid >= (1LL << 31)) {
        set_error("fp8: %lld rows", (long long)rows);
        return EINVAL_ARG;
    }
    const int64_t ld = fp8_row_bytes(K), sld = fp8_row_scales(K);
    if (dtype == BF16) f8_rows<F8BF16><<<(unsigned)grid, 256, 0, st>>>((const uint16_t*)x, rows, (int)K, (int)KB, q, ld, s, sld);
    else f8_rows<F8F16><<<(unsigned)grid, 256, 0, st>>>((const uint16_t*)x, rows, (int)K, (int)KB, q, ld, s, sld);
    KMI_CHECK_LAUNCH("fp8 rows");
    return OK;
}

int launch_fp8_gemm(const F8Args& a, bool glu, int64_t tiles, hipStream_t st) {
    if (glu) return go<HALF, 4, 2, 4, 3, true>(a, tiles, st);
    if (a.tm <= 64) return go<2, 2, 2, 3>(a, tiles, st);
    if (a.tm <= 128) return go<2, 2, 4, 2>(a, tiles, st);
    return go<4, 2, 8, 2>(a, tiles, st);
}

}  // namespace kmi
