// The gate|up products of block-scaled E4M3 experts at prefill sizes: tiles of up to
// 64 rows of one expert x 128 gate and 128 up rows, SwiGLU, and the activations
// quantized for the down product.
//
// What these products are rounded to, E4M3 again, turns a small error of a sum into
// an eighth of a value where a code falls to its neighbour; the 8-bit matrix
// instructions drop too much of small products for that (fp8.hpp).  So the codes
// are multiplied in bfloat16, which holds them exactly: the weights' turned on their
// way from LDS to v_mfma_f32_32x32x16_bf16, x's values (codes times the row's scale, a
// power of two) by the pass before.  The weights' scale joins its codes as a power of
// two (exact), and its mantissa the block's sums, in float32.
//
// 4 waves: 32 gate and 32 up rows x the tile's one or two blocks of 32 rows each.
// A workgroup starts with a chain of latencies (its tile, its rows, their first
// inputs: 4 us) and ends with SwiGLU (5 us) beside some 20 us of products, so two
// of them share a CU: K goes in halves of a block, 64 inputs, 24 KB of LDS each.  A
// lane holds its row's 32 inputs of a half in registers, so the half's place is free
// once they are read, a half ahead: two halves' loads are in flight beside the one
// that has landed.
//
// 16384 rows of 128 experts, 2048 -> 768: 156-188 us (103 GFLOP: 0.66 PFLOP/s of the
// 1.84 that these instructions reach on the whole chip).  Without the products
// 143 us, without the loads 120, without either 104: data and products are of like
// length and hide each other only in part.
#include "fp8_tiles.hpp"

namespace kmi {

namespace {

constexpr int U_TM = 64, U_WAVES = 4, U_STAGES = 3, U_K = 64;          // U_K: inputs of a half
constexpr int U_WTILE = 256 * U_K, U_STAGE = U_WTILE + 2 * U_TM * U_K;
constexpr int U_WL = U_WTILE / 1024 / U_WAVES, U_XL = 2 * U_TM * U_K / 1024 / U_WAVES;  // loads per wave and half
constexpr int U_LDS = U_STAGES * U_STAGE;
constexpr int U_ROW = 272;                                             // bytes of an activation row in LDS, padded

// TAIL: K is not a multiple of 64
template <bool TAIL>
__global__ __launch_bounds__(64 * U_WAVES, 2) void f8_glu(F8Args a, int nblocks, GPlace place, int tiles) {
    extern __shared__ __align__(16) unsigned char smem[];
    const uint32_t lds = g_lds(smem);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, h = lane >> 5;
    int tile, nb;
    g_place((int)blockIdx.x, place, tile, nb);
    if (tile >= tiles || nb >= nblocks) return;
    const GTile T = g_tile(a, tile);
    const int count = T.count;
    if (count <= 0) return;

    const int K = (int)a.K, KB = (K + F8_BLOCK - 1) / F8_BLOCK;
    // the weights' scales, 64 blocks, one per lane (gate, up)
    const int64_t SB = (a.wrows + F8_BLOCK - 1) / F8_BLOCK;
    const int64_t sbase = (T.expert * SB + nb) * KB;
    float swl[2], spl[2];                                     // the scale is swl * spl, spl a power of two
    auto load_scales = [&](int t) {
        const int64_t i = sbase + (t + lane < KB ? t + lane : KB - 1), up = a.N / F8_BLOCK * KB;
        uint32_t v[2];
        if (a.e8) {
            v[0] = ((const unsigned char*)a.s)[i];
            v[1] = ((const unsigned char*)a.s)[i + up];
        } else {
            v[0] = ((const uint32_t*)a.s)[i];
            v[1] = ((const uint32_t*)a.s)[i + up];
        }
        asm volatile("" : "+v"(v[0]), "+v"(v[1]));            // waited for here, not in the loop
#pragma unroll
        for (int g = 0; g < 2; g++) {
            uint32_t e;
            f8_split(a.e8 ? e8m0_to_f32(v[g]) : __uint_as_float(v[g]), e, swl[g]);
            // no further than bfloat16 holds a code's multiple; past that, none of
            // the rest leaves float32's range that the result does not
            const uint32_t in = e < 63 ? 63 : e > 191 ? 191 : e;
            swl[g] = __builtin_amdgcn_ldexpf(swl[g], (int)e - (int)in);
            spl[g] = __uint_as_float(in << 23);
        }
    };
    int64_t xr[U_XL];                                         // (beside the scales' latency)
    g_xrows(a, T, 8 * wave + (lane >> 3), 8 * U_WAVES, xr);
    load_scales(0);
    // direct-to-LDS loads: 4 lanes per weight row of 64 bytes, 8 per x row of 128, the
    // lane's piece permuted by the row, so that 8 rows' reads fall on distinct banks;
    // LDS weight row 64 v + r: gate row 32 v + r of the block, r < 32, or up row.
    // (From here on the compiler's counts miss what is in flight: no load that it
    // would wait for.)
    const int piece = (lane & 3) ^ (lane >> 3 & 3);           // (row / 2 % 4 == lane / 8 % 4)
    const int64_t n0 = (int64_t)nb * 128;                     // N is a multiple of 128
    const unsigned char* const xv = (const unsigned char*)a.x;
    const unsigned char* const wv = a.w + (T.expert * a.wrows + n0 + (wave & 2 ? a.N : 0)) * a.K;     // (a wave loads gate or up rows)
    const int64_t xbytes = a.xrows * a.xld, wbytes = 128 * a.K;
    uint32_t xoff[U_XL], woff[U_WL];
#pragma unroll
    for (int j = 0; j < U_XL; j++) {
        xoff[j] = xr[j] < 0 ? G_NONE : (uint32_t)(xr[j] * a.xld) + 16u * ((lane & 7) ^ (lane >> 3));
    }
#pragma unroll
    for (int j = 0; j < U_WL; j++) {
        const int m = 16 * (wave + U_WAVES * j) + (lane >> 2);
        woff[j] = (uint32_t)((m >> 6) * 32 + (m & 31)) * (uint32_t)K + 16u * piece;
    }
    auto issue = [&](int t, int at) {                         // half t (past the last: zeros) into place `at`
        const bool on = t * U_K < K;
        const __amdgpu_buffer_rsrc_t rw = make_rsrc(wv, on ? wbytes : 0), rx = make_rsrc(xv, on ? xbytes : 0);
        const uint32_t dst = lds + at * U_STAGE + wave * 1024;
        const bool in = !TAIL || t * U_K + 16 * piece < K;    // inputs past the last: zeros
#pragma unroll
        for (int j = 0; j < U_WL; j++)
            g_dma16(rw, dst + U_WAVES * j * 1024, in ? woff[j] : G_NONE, (uint32_t)t * U_K);
#pragma unroll
        for (int j = 0; j < U_XL; j++)
            g_dma16(rx, dst + U_WTILE + U_WAVES * j * 1024, xoff[j], (uint32_t)t * U_K * 2);
    };
#pragma unroll
    for (int t = 0; t < U_STAGES; t++) issue(t, t);

    // this lane's row of fragment i (weights) or j (x): inputs 32 h .. of a half, in
    // 16-byte pieces 2 h + q (x: 4 h + s)
    uint32_t wo[2], xo[4];
#pragma unroll
    for (int q = 0; q < 2; q++) wo[q] = (uint32_t)(64 * wave + l32) * U_K + 16u * ((2 * h + q) ^ (l32 >> 1 & 3));
#pragma unroll
    for (int s = 0; s < 4; s++) xo[s] = U_WTILE + (uint32_t)l32 * 2 * U_K + 16u * ((4 * h + s) ^ (l32 & 7));
    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[i][j][r] = 0.f;

    // NJ: the tile's blocks of 32 rows
    auto run = [&](auto nj) {
        constexpr int NJ = decltype(nj)::value;
        u32x4 w[2][2];
        bf16x8 x[NJ][4];
        // the operands of step s (weights: of two) of the half at place `at`
        auto read = [&](int at, int s) {
            const unsigned char* st = smem + at * U_STAGE;
            if (s % 2)
#pragma unroll
                for (int i = 0; i < 2; i++) w[i][s / 2] = *(const u32x4*)(st + i * 32 * U_K + wo[s / 2]);
#pragma unroll
            for (int j = 0; j < NJ; j++) x[j][s] = *(const bf16x8*)(st + j * 64 * U_K + xo[s]);
        };
        g_wait<(U_STAGES - 1) * (U_WL + U_XL)>();
        lds_barrier();
#pragma unroll
        for (int s = 0; s < 4; s++) read(0, s);
        int at = 0;                                           // this half's place in the ring
        for (int t0 = 0; t0 < KB; t0 += G_CHUNK) {
            if (t0) load_scales(t0);
            const int t1 = t0 + G_CHUNK < KB ? t0 + G_CHUNK : KB;
            for (int t = t0; t < t1; t++) {
                f32x16 p[2][NJ];
                float sp[2];
#pragma unroll
                for (int i = 0; i < 2; i++)
                    sp[i] = __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(spl[i]), t % G_CHUNK));
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int j = 0; j < NJ; j++)
#pragma unroll
                        for (int r = 0; r < 16; r++) p[i][j][r] = 0.f;
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    // this half is in registers everywhere and the next one has landed
                    g_wait<(U_STAGES - 2) * (U_WL + U_XL)>();
                    lds_barrier();
                    issue(2 * t + half + U_STAGES, at);
                    at = at + 1 < U_STAGES ? at + 1 : 0;
#pragma unroll
                    for (int s = 0; s < 4; s++) {
                        bf16x8 wv[2];
#pragma unroll
                        for (int i = 0; i < 2; i++) wv[i] = f8_values(w[i][s / 2][s % 2 * 2], w[i][s / 2][s % 2 * 2 + 1], sp[i]);
#pragma unroll
                        for (int i = 0; i < 2; i++)
#pragma unroll
                            for (int j = 0; j < NJ; j++)
                                p[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wv[i], x[j][s], p[i][j], 0, 0, 0);
                        read(at, s);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float sw = __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(swl[i]), t % G_CHUNK));
#pragma unroll
                    for (int j = 0; j < NJ; j++)
#pragma unroll
                        for (int r = 0; r < 16; r++) acc[i][j][r] = __builtin_fmaf(p[i][j][r], sw, acc[i][j][r]);
                }
            }
        }
    };
    const int nj = (count + 31) / 32;
    if (nj == 2) run(std::integral_constant<int, 2>());
    else run(std::integral_constant<int, 1>());
    g_wait<0>();                                 // no load still writes LDS below
    lds_barrier();

    // activations of 128 columns per row through LDS, where 16 lanes quantize a
    // row's group.  D: row 8 (r / 4) + 4 h + r % 4 of the fragment, x row l % 32
#pragma unroll
    for (int j = 0; j < 2; j++) {
        if (j >= nj) break;
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            uint32_t o[2];
#pragma unroll
            for (int q = 0; q < 2; q++) {
                const uint32_t g = cvt_pk_bf16(acc[0][j][r + 2 * q], acc[0][j][r + 2 * q + 1]);
                const uint32_t u = cvt_pk_bf16(acc[1][j][r + 2 * q], acc[1][j][r + 2 * q + 1]);
                o[q] = cvt_pk_bf16(silu_bf16r(__uint_as_float(g << 16)) * __uint_as_float(u << 16),
                                   silu_bf16r(__uint_as_float(g & 0xffff0000u)) * __uint_as_float(u & 0xffff0000u));
            }
            *(u32x2*)(smem + (32 * j + l32) * U_ROW + (32 * wave + 2 * r + 4 * h) * 2) = u32x2{o[0], o[1]};
        }
    }
    lds_barrier();
    const int l16 = tid & 15;
    for (int m = tid >> 4; m < count; m += 4 * U_WAVES) {
        F8Raw<F8BF16, 8> v;
        v.v[0] = *(const u32x4*)(smem + m * U_ROW + 16 * l16);
        uint32_t byte = f8_scale_byte(f8_max16(v.amax()));
        const bool nan = byte == 255;            // as f8_rows
        if (nan) byte = 127;
        const float scale = __uint_as_float(byte << 23);
        unsigned char* y = (unsigned char*)a.y + (T.start + m) * a.N + nb * 128 + 8 * l16;
        *(u32x2*)y = nan ? u32x2{0x7f7f7f7fu, 0x7f7f7f7fu} : u32x2{v.codes(0, scale), v.codes(1, scale)};
        if (l16 == 0) a.ys[(T.start + m) * a.ys_ld + nb] = (unsigned char)byte;
    }
}

}  // namespace

int launch_fp8_glu(const F8Args& a, int64_t tiles, hipStream_t st) {
    if (!a.tiles || a.K > FP8_GEMM_MAX_K || a.xld != 2 * fp8_row_bytes(a.K) || a.tm != U_TM || a.N % 128 ||
        a.xrows * a.xld >= (1LL << 31)) {
        set_error("fp8: gate|up tiles of %d rows, K=%lld, N=%lld", a.tm, (long long)a.K, (long long)a.N);
        return EINVAL_ARG;
    }
    const int64_t nblocks = a.N / 128;
    const GPlace place = g_place_of(nblocks);
    const int64_t wgs = g_place_grid(tiles, place);
    if (wgs >= (1LL << 31)) {
        set_error("fp8: grid of %lld workgroups", (long long)wgs);
        return EINVAL_ARG;
    }
    const auto f = a.K % U_K ? f8_glu<true> : f8_glu<false>;
    allow_dynamic_lds_once((const void*)f);
    f<<<(unsigned)wgs, 64 * U_WAVES, U_LDS, st>>>(a, (int)nblocks, place, (int)tiles);
    KMI_CHECK_LAUNCH("fp8 gate|up");
    return OK;
}

}  // namespace kmi
