// Block-scaled E4M3 products of many rows: tiles of 128 or 256 weight rows x 64 to
// 256 activation rows.
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
//
// Bound by the matrix instructions in full tiles: 4096 rows of [4096, 14336] 185 us
// (2.6 PFLOP/s; the chip gives an 8-bit 16 x 16 x 128 every 32 cycles at 2.16 GHz,
// 175 us) and 35 of the pass before, called now and then; call after call the same tiles
// take 196-229.  2048 rows of [14336, 4096] are 448 tiles on 256 CUs, 1.75 rounds:
// 131 us + 8.  Few rows are bound by a workgroup's chain of latencies: 77 rows of
// [4100, 2064] 12 us + 3; rows of many experts by the weights' stream: 128 rows that
// reach 62 of 128 experts [1536, 2048] (197 MB) 39-43 us, 4.6-5.0 TB/s, + 5 for the sort
// and 3 for x.
#include "fp8_tiles.hpp"

namespace kmi {

namespace {

// how the scales meet the sums: powers of two by the instruction, and float32
// scales' mantissas after it, in float32, block by block
enum Kind { F32S, E8S };

// NW x WM waves: 64 weight rows x MB 16-row blocks of activations each
template <int NW, int WM, int MB, int S>
struct Shape {
    static constexpr int TN = 64 * NW, TM = 16 * MB * WM, WAVES = NW * WM;
    static constexpr int WTILE = TN * F8_BLOCK, STAGE = WTILE + TM * F8_BLOCK;   // a block's bytes in LDS
    static constexpr int XL = TM / 8 / WAVES, WL = TN / 8 / WAVES;               // loads per wave and block
    static constexpr int LDS = S * STAGE + G_CHUNK * TM;
    static_assert(XL * 8 * WAVES == TM && WL * 8 * WAVES == TN, "whole loads per wave");
};

// TAIL: K is not a multiple of 128; MANY: several column blocks per workgroup;
// PART: blocks [per z, per z + per) of K (grid z), sums to a.partial
template <Kind KIND, int NW, int WM, int MB, int S, bool TAIL, bool MANY, bool PART>
__global__ __launch_bounds__(64 * NW * WM, 2) void f8_gemm(F8Args a, int nblocks, GPlace place, int tiles, int many, int per) {
    typedef Shape<NW, WM, MB, S> Z;
    constexpr int RB = 4, TN = Z::TN, TM = Z::TM, XL = Z::XL, WL = Z::WL, WAVES = Z::WAVES, WTILE = Z::WTILE;
    static_assert(!MANY || S == 2, "stores among the loads in flight: their wait is for all of them");
    const int nl = MANY ? many : 1;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int rid_s[TM];
    unsigned char* const sc = smem + S * Z::STAGE;            // [G_CHUNK / 16][TM][16] scale bytes
    const uint32_t lds = g_lds(smem), lds_sc = lds + S * Z::STAGE;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave % NW, wm = wave / NW;
    const int l16 = lane & 15, c = lane >> 4;
    // workgroup -> (tile, nl column blocks from nb nl): grouped as g_place; dense, each XCD takes
    // an eighth of the pairs, in strips of 8 tiles (weights and x shared in its L2)
    int tile, nb;
    if (a.tiles) {
        g_place((int)blockIdx.x, place, tile, nb);
        if (tile >= tiles || nb >= nblocks) return;
    } else {
        const int xcd = (int)blockIdx.x & 7, kk = (int)blockIdx.x >> 3;
        const int idx = xcd * ((int)gridDim.x >> 3) + kk, strip = idx / (8 * nblocks), in = idx - strip * 8 * nblocks;
        if (idx >= tiles * nblocks) return;
        const int height = tiles - 8 * strip < 8 ? tiles - 8 * strip : 8;
        tile = 8 * strip + in % height;
        nb = in / height;
    }
    const GTile T = g_tile(a, tile);
    const int count = T.count;
    if (count <= 0) return;

    const int K = (int)a.K, KBs = (K + F8_BLOCK - 1) / F8_BLOCK;
    const int kb0 = PART ? (int)blockIdx.y * per : 0, KB = PART ? KBs - kb0 < per ? KBs - kb0 : per : KBs;
    if (PART) a.xs += kb0;
    const int64_t x0 = a.tiles ? 0 : T.start;                 // the x view's first row
    // the weights' scales of the wave's rows, 64 blocks, one per lane
    // (several column blocks: KB nl <= 64, all of theirs)
    const int64_t first = (int64_t)nb * nl * TN;              // the first column
    const int64_t SB = (a.wrows + F8_BLOCK - 1) / F8_BLOCK;
    uint32_t swl;                                // the scale's byte
    float sml = 1.f;                             // and its mantissa (F32S)
    auto load_scales = [&](int t) {
        int kb = t + lane, b = 0;
        if (MANY) {
            b = kb / KB;
            kb -= b * KB;
        }
        const int64_t n = first + (int64_t)b * TN + 64 * wn;
        const int64_t i = (T.expert * SB + (n < a.N ? n : first) / F8_BLOCK) * KBs + kb0 + (kb < KB ? kb : KB - 1);
        if (KIND == E8S) swl = ((const unsigned char*)a.s)[i];
        else f8_split(((const float*)a.s)[i], swl, sml);
        asm volatile("" : "+v"(swl), "+v"(sml));              // waited for here, not in the loop
    };
    int64_t xr[XL];                                           // (beside the scales' latency)
    g_xrows(a, T, 8 * wave + (lane >> 3), 8 * WAVES, xr);
    load_scales(0);
    if (tid < TM) rid_s[tid] = tid >= count ? -1 : a.tiles ? a.sorted[T.start + tid] : (int)(T.start + tid);
    // direct-to-LDS loads: 8 lanes per row, the lane's piece permuted by the row.
    // (From here on the compiler's counts miss what is in flight: no load that it
    // would wait for.)
    const int piece = (lane & 7) ^ (lane >> 3);               // (row % 8 == lane / 8)
    const int k0 = kb0 * F8_BLOCK;
    const unsigned char* const xv = (const unsigned char*)a.x + x0 * a.xld + k0;
    const int64_t xbytes = (a.xrows - x0) * a.xld - k0;
    uint32_t xoff[XL], woff[WL];
#pragma unroll
    for (int j = 0; j < XL; j++) {
        xoff[j] = xr[j] < 0 ? G_NONE : (uint32_t)((xr[j] - x0) * a.xld) + 16u * piece;
    }
#pragma unroll
    for (int j = 0; j < WL; j++) {
        woff[j] = (uint32_t)(8 * (wave + WAVES * j) + (lane >> 3)) * (uint32_t)K + 16u * piece;   // (past the view: zeros)
    }
    // the next block in turn, of this column block or the next (past the last: zeros)
    int it = 0, rows = (int)(a.N - first < (int64_t)nl * TN ? a.N - first : (int64_t)nl * TN);
    const unsigned char* wv = a.w + (T.expert * a.wrows + first) * a.K + k0;
    auto issue = [&](int at) {
        const __amdgpu_buffer_rsrc_t rw = make_rsrc(wv, rows > 0 ? (rows < TN ? rows : TN) * K - k0 : 0);
        const __amdgpu_buffer_rsrc_t rx = make_rsrc(xv, rows > 0 ? xbytes : 0);
        const uint32_t dst = lds + at * Z::STAGE + wave * 1024;
        const bool in = !TAIL || k0 + it * F8_BLOCK + 16 * piece < K;      // inputs past the last: zeros
#pragma unroll
        for (int j = 0; j < WL; j++)
            g_dma16(rw, dst + WAVES * j * 1024, in ? woff[j] : G_NONE, (uint32_t)it * F8_BLOCK);
#pragma unroll
        for (int j = 0; j < XL; j++) g_dma16(rx, dst + WTILE + WAVES * j * 1024, xoff[j], (uint32_t)it * F8_BLOCK);
        it = it + 1 < KB ? it + 1 : 0;
        rows -= it ? 0 : TN;
        wv += it ? 0 : TN * K;                                // (not read past the last)
    };
    g_scales<TM, WAVES>(a, T, lds_sc, 0, KB, wave, lane);
#pragma unroll
    for (int t = 0; t < S; t++) issue(t);

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
    g_wait<(S - 1) * (XL + WL)>();
    lds_barrier();
#pragma unroll
    for (int i = 0; i < RB; i++) read_w(smem, i);
    read_b(smem, 0);
    static_assert(MB % 2 == 0, "x fragments alternate");
    int at = 0;                                  // this block's place in the ring
    for (int cb = 0; cb < nl; cb++) {
    const int64_t n0 = first + (int64_t)cb * TN;
    if (n0 >= a.N) break;
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int j = 0; j < MB; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int t0 = 0; t0 < KB; t0 += G_CHUNK) {
    if (t0) {                                    // every wave is past its reads of the last chunk's scales
        load_scales(t0);
        g_scales<TM, WAVES>(a, T, lds_sc, t0, KB, wave, lane);
        g_wait<0>();
        lds_barrier();
    }
    const int t1 = t0 + G_CHUNK < KB ? t0 + G_CHUNK : KB;
    for (int t = t0; t < t1; t++) {              // (no branch inside: the compiler would sink products past it)
        const int after = at + 1 < S ? at + 1 : 0;
        const unsigned char* st = smem + at * Z::STAGE;
        const unsigned char* nx = smem + after * Z::STAGE;
        uint32_t sx[MB];
#pragma unroll
        for (int j = 0; j < MB; j++) sx[j] = g_scale(sc, TM, 16 * (MB * wm + j) + l16, t);
        const uint32_t sw = (uint32_t)__builtin_amdgcn_readlane((int)swl, (cb * KB + t) % G_CHUNK);
        const float sm = __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(sml), (cb * KB + t) % G_CHUNK));
        // after the block's last LDS read: the next block has landed, and this
        // one's place is free
        auto turn = [&]() {
            g_wait<(S - 2) * (XL + WL)>();
            lds_barrier();
            issue(at);
        };
        {
            // product n = 4 j + i; its sums meet the mantissa two products later
            constexpr int NP = RB * MB;
            f32x4 p[3];
            auto apply = [&](int n) {
                const int i = n % RB, j = n / RB;
#pragma unroll
                for (int q = 0; q < 4; q++) acc[i][j][q] = __builtin_fmaf(p[n % 3][q], sm, acc[i][j][q]);
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
                    acc[i][j] = f8_mfma(w[i], b[j & 1], acc[i][j], sw, sx[j]);
                } else {
                    p[n % 3] = f8_mfma(w[i], b[j & 1], f32x4{0.f, 0.f, 0.f, 0.f}, sw, sx[j]);
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
        at = after;
    }
    }
    {
        uint16_t* y = (uint16_t*)a.y;
        const bool wide = a.N % 4 == 0 && ((uintptr_t)a.y & 7) == 0;
#pragma unroll
        for (int j = 0; j < MB; j++) {
            const int m = 16 * (MB * wm + j) + l16;
            const int rid = rid_s[m];
            if (rid < 0) continue;
            bool seen = true;
            if (a.lhs) {
                int64_t row[1];
                g_xrows(a, T, m, 0, row);
                seen = row[0] >= 0;
            }
#pragma unroll
            for (int i = 0; i < RB; i++) {
                const int64_t n = n0 + 64 * wn + 16 * i + 4 * c;
                if constexpr (PART) {            // rows of whole blocks of 4
                    if (n < a.N) *(f32x4*)(a.partial + ((int64_t)blockIdx.y * a.rows + rid) * a.part_ld + n) = acc[i][j];
                    continue;
                }
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
    g_wait<0>();                                 // no load still writes LDS when the workgroup ends
}

// y[m, n] = the parts' sums, in order, rounded once: 4 columns per thread
__global__ __launch_bounds__(256) void f8_reduce(const float* __restrict__ part, int parts, int64_t rows, int64_t ld,
                                                 int64_t N, int half, uint16_t* __restrict__ y) {
    const int64_t per = ld / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * per) return;
    const int64_t m = i / per, n = i % per * 4;
    f32x4 v = *(const f32x4*)(part + m * ld + n);
    for (int p = 1; p < parts; p++) {
        const f32x4 o = *(const f32x4*)(part + (p * rows + m) * ld + n);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += o[e];
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (n + e < N) y[m * N + n + e] = half ? f32_to_f16(v[e]) : f32_to_bf16(v[e]);
}

// x's rows into codes [rows, ld] (tails zero) and scale bytes [rows, sld]: 16
// lanes per row and block.  VALUES: what they stand for, in bfloat16, instead.
template <class T, bool VALUES>
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
    const u32x2 c = nan ? u32x2{0x7f7f7f7fu, 0x7f7f7f7fu} : u32x2{v.codes(0, scale), v.codes(1, scale)};
    if constexpr (VALUES) {
        *(bf16x8*)(q + r * ld + 2 * k) = f8_values(c.x, c.y, scale);
        return;
    }
    *(u32x2*)(q + r * ld + k) = c;
    if (l == 0) s[r * sld + b] = (unsigned char)byte;
}

template <Kind KIND, int NW, int WM, int MB, int S, bool TAIL, bool MANY, bool PART>
int go(const F8Args& a, int64_t tiles, int parts, hipStream_t st) {
    typedef Shape<NW, WM, MB, S> Z;
    if (a.K > FP8_GEMM_MAX_K || a.xld != fp8_row_bytes(a.K) || a.tm > Z::TM) {
        set_error("fp8: K=%lld in tiles of %d", (long long)a.K, a.tm);
        return EINVAL_ARG;
    }
    // Column blocks per workgroup.  A workgroup's start (its tile, its rows, their
    // first inputs) takes as long as some ten blocks of K, so a short K takes
    // several column blocks, their weights streaming on, while the grid keeps twice
    // what runs at once (the expert block of 2048 tokens, down [2048, 768]: 2 or 4 blocks
    // 271 us, 1 278, 8 285); so does any K where most of a tile is empty, and the weights' stream is
    // all there is, while two workgroups come to a CU (512 rows of 64 experts
    // [2048, 2048]: 2 blocks 61.9 us, 1 65.7, 4 78.0; 4096 rows: 88.2, 89.1, 101.8).
    const int64_t KB = ceil_div(a.K, F8_BLOCK);
    int many = 1;
    if (MANY) {
        const int64_t experts = a.E < a.rows ? a.E : a.rows, some = ceil_div(a.rows, a.tm) + experts / 2;
        const int64_t active = some > experts ? some : experts;
        while (2 * many * KB <= 24 && active * ceil_div(a.N, 2 * many * Z::TN) >= 1536) many *= 2;
        if (many == 1 && 2 * KB <= G_CHUNK && a.rows < 64 * a.E && active * ceil_div(a.N, 2 * Z::TN) >= 512) many = 2;
    }
    const int nblocks = (int)ceil_div(a.N, (int64_t)many * Z::TN);
    const GPlace place = g_place_of(nblocks);
    const int64_t wgs = a.tiles ? g_place_grid(tiles, place) : ceil_div(tiles * nblocks, 8) * 8;
    if (wgs >= (1LL << 31)) {
        set_error("fp8: grid of %lld workgroups", (long long)wgs);
        return EINVAL_ARG;
    }
    const auto f = f8_gemm<KIND, NW, WM, MB, S, TAIL, MANY, PART>;
    allow_dynamic_lds_once((const void*)f);
    const int per = PART ? fp8_part_blocks(a.K, parts) : 0;
    f<<<dim3((unsigned)wgs, (unsigned)parts), 64 * Z::WAVES, Z::LDS, st>>>(a, nblocks, place, (int)tiles, many, per);
    KMI_CHECK_LAUNCH("fp8 tiles");
    if (PART) {
        const int64_t n = ceil_div(a.rows * (a.part_ld / 4), 256);
        f8_reduce<<<(unsigned)n, 256, 0, st>>>(a.partial, parts, a.rows, a.part_ld, a.N, a.half, (uint16_t*)a.y);
        KMI_CHECK_LAUNCH("fp8 parts");
    }
    return OK;
}

template <int NW, int WM, int MB, int S, bool MANY, bool PART>
int go(const F8Args& a, int64_t tiles, int parts, hipStream_t st) {
    if (a.K % F8_BLOCK)
        return a.e8 ? go<E8S, NW, WM, MB, S, true, MANY, PART>(a, tiles, parts, st)
                    : go<F32S, NW, WM, MB, S, true, MANY, PART>(a, tiles, parts, st);
    return a.e8 ? go<E8S, NW, WM, MB, S, false, MANY, PART>(a, tiles, parts, st)
                : go<F32S, NW, WM, MB, S, false, MANY, PART>(a, tiles, parts, st);
}

}  // namespace

int64_t fp8_row_bytes(int64_t K) { return ceil_div(K, F8_BLOCK) * F8_BLOCK; }
int64_t fp8_row_scales(int64_t K) { return ceil_div(ceil_div(K, F8_BLOCK), 16) * 16; }

int launch_fp8_rows(const void* x, int dtype, int64_t rows, int64_t K, unsigned char* q, unsigned char* s,
                    hipStream_t st) {
    const int64_t KB = ceil_div(K, F8_BLOCK), grid = ceil_div(rows * KB, 16);
    if (grid >= (1LL << 31)) {
        set_error("fp8: %lld rows", (long long)rows);
        return EINVAL_ARG;
    }
    const int64_t ld = fp8_row_bytes(K) * (s ? 1 : 2), sld = fp8_row_scales(K);
    const auto f = dtype == BF16 ? s ? f8_rows<F8BF16, false> : f8_rows<F8BF16, true>
                                 : s ? f8_rows<F8F16, false> : f8_rows<F8F16, true>;
    f<<<(unsigned)grid, 256, 0, st>>>((const uint16_t*)x, rows, (int)K, (int)KB, q, ld, s, sld);
    KMI_CHECK_LAUNCH("fp8 rows");
    return OK;
}

int fp8_part_blocks(int64_t K, int parts) {
    return (int)(ceil_div(ceil_div(ceil_div(K, F8_BLOCK), parts), 4) * 4);       // (scale bytes in words)
}

// Dense products of few tiles split K into parts of at least 8 blocks, while a CU
// has no workgroup.  [4096, 14336] x 33 rows (32 tiles): 8 parts 22.5 us, 4 27.0,
// whole 56.1; [14336, 4096] x 64 (112): 2 parts 23.9, 4 28.0, whole 26.0; [4096,
// 4096] x 256 (128): 2 parts 22.0, whole 21.7.  A K of 17 blocks: 2 parts 14.4,
// whole 14.2.
int fp8_gemm_parts(int64_t M, int64_t K, int64_t N, int tm) {
    const int64_t wgs = ceil_div(M, tm) * ceil_div(N, 128), KB = ceil_div(K, F8_BLOCK);
    if (tm > 64 || KB < 32) return 1;
    const int64_t idle = 256 / wgs, most = KB / 8;
    const int parts = (int)(idle < most ? idle : most);
    return parts < 2 ? 1 : (int)ceil_div(KB, fp8_part_blocks(K, parts));
}

int launch_fp8_gemm(const F8Args& a, int64_t tiles, int parts, hipStream_t st) {
    if (a.tiles) return a.tm <= 64 ? go<2, 2, 2, 2, true, false>(a, tiles, 1, st) : go<2, 2, 4, 2, true, false>(a, tiles, 1, st);
    if (parts > 1) return go<2, 2, 2, 3, false, true>(a, tiles, parts, st);
    if (a.tm <= 64) return go<2, 2, 2, 3, false, false>(a, tiles, 1, st);
    if (a.tm <= 128) return go<2, 2, 4, 2, false, false>(a, tiles, 1, st);
    return go<4, 2, 8, 2, false, false>(a, tiles, 1, st);
}

}  // namespace kmi
