// Block-scaled E4M3 products of many rows, on tiles of 256 weight rows x up to
// 128 activation rows (gate|up: 128 gate and 128 up rows x up to 64).
//
// The rows of x are quantized by a pass before (fp8_rows).  A workgroup's 4
// waves take 64 weight rows each and all of the tile's activation rows: weights
// go from memory into the matrix operand as they are, one 128-input block
// ahead, and only x, which every wave reads, passes through LDS (direct-to-LDS
// loads, one block ahead; rows of 128 bytes with their 16-byte pieces permuted
// by the row, so 8 rows' reads fall on distinct banks).  D holds activation rows
// along its columns, so a lane has one row's scale per 16 x 16 tile.
#include "fp8.hpp"

namespace kmi {

namespace {

#define KMI_F8_LDS(p) ((__attribute__((address_space(3))) void*)(p))

constexpr int G_WAVES = 4;
constexpr int G_STAGES = 2;
constexpr uint32_t G_NONE = 0x80000000u;     // past every view: reads 0

// how weights and x meet: E4M3 operands with both scales applied to each
// block's sums in float32 (weights' scales in float32), or by the instruction
// (E8M0); or float16 operands (gate|up, whose results are rounded to E4M3 again)
enum Kind { F32S, E8S, HALF };

template <int N_>
__device__ __forceinline__ void g_wait() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N_) : "memory");
}

// 16 bytes per lane from the view's offset into LDS at dst + 16 lane.  In asm, as
// the compiler would wait for the load before any later read of LDS; the kernel
// waits for it itself (g_wait), and its own counts, which miss these loads, only
// wait for more.
__device__ __forceinline__ void g_dma16(__amdgpu_buffer_rsrc_t r, unsigned char* dst, uint32_t voff, uint32_t soff) {
    const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)dst;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 ::"s"(at), "v"(voff), "s"(r), "s"(soff) : "memory", "m0");
}

template <int MB, Kind KIND, bool GLU>
__global__ __launch_bounds__(64 * G_WAVES, 2) void f8_gemm(F8Args a, int nblocks, int tiles) {
    constexpr int TM = 16 * MB, RB = 4;
    constexpr int XB = KIND == HALF ? 256 : 128;              // bytes of a row's block in LDS
    constexpr int PER = TM * XB / 1024 / G_WAVES;             // direct-to-LDS loads per wave and block
    constexpr int STAGE = TM * XB;
    static_assert(PER * 1024 * G_WAVES == STAGE, "whole loads per wave");
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int rid_s[TM];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
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
    const int64_t xld = a.xld;                                // bytes per x row
    // x rows of the tile; its view starts at row x0
    const int64_t x0 = a.tiles ? 0 : start;
    unsigned char* sc = smem + G_STAGES * STAGE;              // [KB][16][8] scale bytes
    auto xrow = [&](int m) -> int64_t {                       // x row of tile row m, or -1
        if (m >= count) return -1;
        if (!a.tiles) return start + m;
        const int rid = a.sorted[start + m];
        const int p = rid / (int)a.Mper;
        const int64_t b = a.lhs ? a.lhs[p] : p / (int)a.lhs_div;
        const int64_t r = b * a.Mper + rid % (int)a.Mper;
        return b >= 0 && r < a.xrows ? r : -1;
    };
    const __amdgpu_buffer_rsrc_t rx = make_rsrc((const unsigned char*)a.x + x0 * xld, (a.xrows - x0) * xld);
    uint32_t xoff[PER];
#pragma unroll
    for (int j = 0; j < PER; j++) {
        constexpr int LPR = XB / 16;                          // lanes per row
        const int m = (64 / LPR) * (wave + G_WAVES * j) + lane / LPR;
        const int64_t r = xrow(m);
        xoff[j] = r < 0 ? G_NONE : (uint32_t)((r - x0) * xld) + 16u * ((lane % LPR) ^ (m & 7));
    }
    auto issue_x = [&](int t) {
        unsigned char* dst = smem + (t & 1) * STAGE;
#pragma unroll
        for (int j = 0; j < PER; j++)
            g_dma16(rx, dst + (wave + G_WAVES * j) * 1024, t < KB ? xoff[j] : G_NONE, (uint32_t)t * XB);
    };
    // a wave's weights: rows 16 i + l16 of its 64 (gate|up: fragments 0, 1 of the
    // gate rows, 2, 3 of the up rows); rows past the last read zeros
    const int64_t n0 = GLU ? (int64_t)nb * 128 + 32 * wave : (int64_t)nb * 256 + 64 * wave;
    const int64_t SB = (a.wrows + F8_BLOCK - 1) / F8_BLOCK;
    int64_t left = a.N - n0;
    left = left < 0 ? 0 : left > (GLU ? 32 : 64) ? (GLU ? 32 : 64) : left;
    const unsigned char* wbase = a.w + (expert * a.wrows + (left ? n0 : 0)) * a.K;
    const __amdgpu_buffer_rsrc_t rw = make_rsrc(wbase, left * a.K);
    const __amdgpu_buffer_rsrc_t ru = make_rsrc(wbase + (GLU ? a.N * a.K : 0), left * a.K);
    uint32_t woff[RB];
#pragma unroll
    for (int i = 0; i < RB; i++) woff[i] = (uint32_t)(16 * (GLU ? i & 1 : i) + l16) * (uint32_t)K + 16u * c;
    u32x4 wn[RB][2];
    auto load_w = [&](int t) {
        const uint32_t k = (uint32_t)(t < KB ? t : KB - 1) * F8_BLOCK;
#pragma unroll
        for (int i = 0; i < RB; i++)
#pragma unroll
            for (int h = 0; h < 2; h++)
                wn[i][h] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                    GLU && i >= 2 ? ru : rw, (int)(woff[i] + k + 64 * h), 0, 0));
    };
    // the weights' scales of 64 blocks, one per lane (gate|up: gate, up)
    const int64_t sbase = (expert * SB + (left ? n0 : 0) / F8_BLOCK) * KB;
    uint32_t swl[GLU ? 2 : 1];
    auto load_s = [&](int t) {
        const int k = t + lane < KB ? t + lane : KB - 1;
#pragma unroll
        for (int g = 0; g < (GLU ? 2 : 1); g++) {
            const int64_t i = sbase + (g ? a.N / F8_BLOCK * KB : 0) + k;
            if (KIND == E8S) swl[g] = ((const unsigned char*)a.s)[i];
            else if (a.e8) swl[g] = __float_as_uint(e8m0_to_f32(((const unsigned char*)a.s)[i]));
            else swl[g] = ((const uint32_t*)a.s)[i];
        }
    };
    issue_x(0);
    load_w(0);
    if (tid < TM) rid_s[tid] = tid >= count ? -1 : a.tiles ? a.sorted[start + tid] : (int)(start + tid);
    // scale bytes of activation row 16 j + n at [block][n][j]
    for (int m = tid & (TM - 1), q = tid / TM; 4 * q < KB; q += 64 * G_WAVES / TM) {
        const int64_t r = xrow(m);
        const uint32_t v = r < 0 ? 0x7f7f7f7fu : *(const uint32_t*)(a.xs + r * a.xs_ld + 4 * q);
#pragma unroll
        for (int b = 0; b < 4; b++)
            if (4 * q + b < KB) sc[((4 * q + b) * 16 + (m & 15)) * 8 + (m >> 4)] = (unsigned char)(v >> (8 * b));
    }

    f32x4 acc[RB][MB];
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int j = 0; j < MB; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // x fragment j: row 16 j + l16, pieces c and c + 4 (float16: 2 c, 2 c + 1 and
    // 8 further)
    uint32_t xo[XB / 64];
#pragma unroll
    for (int q = 0; q < XB / 64; q++) {
        const int piece = KIND == HALF ? 2 * c + (q & 1) + 8 * (q >> 1) : c + 4 * q;
        xo[q] = (uint32_t)l16 * XB + 16u * (piece ^ (l16 & 7));
    }

    for (int t = 0; t < KB; t++) {
        if ((t & 63) == 0) load_s(t);
        // what the block before asked for has landed: this block's x and weights
        g_wait<0>();
#pragma unroll
        for (int i = 0; i < RB; i++) asm volatile("" : "+v"(wn[i][0]), "+v"(wn[i][1]));
        lds_barrier();
        u32x4 w[RB][2];
#pragma unroll
        for (int i = 0; i < RB; i++) {
            w[i][0] = wn[i][0];
            w[i][1] = wn[i][1];
        }
        load_w(t + 1);
        issue_x(t + 1);
        if (t == KB - 1 && K % F8_BLOCK) {       // inputs past the last: the next row's
#pragma unroll
            for (int i = 0; i < RB; i++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                    if (64 * h + 16 * c >= K % F8_BLOCK) w[i][h] = u32x4{0, 0, 0, 0};
        }
        __builtin_amdgcn_sched_barrier(0);
        const unsigned char* xs = smem + (t & 1) * STAGE;
        const u32x2 sx = *(const u32x2*)(sc + (t * 16 + l16) * 8);
        uint32_t sw[GLU ? 2 : 1];
#pragma unroll
        for (int g = 0; g < (GLU ? 2 : 1); g++) sw[g] = (uint32_t)__builtin_amdgcn_readlane((int)swl[g], t & 63);
        auto row_scale = [&](int j) { return __uint_as_float(((j < 4 ? sx.x : sx.y) >> (8 * (j & 3)) & 0xffu) << 23); };
        if constexpr (KIND == HALF) {
            typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
            f16x8 wh[RB][4];
#pragma unroll
            for (int i = 0; i < RB; i++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const uint32_t d0 = w[i][q >> 1][(q & 1) * 2], d1 = w[i][q >> 1][(q & 1) * 2 + 1];
                    const f16x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d0, 1.f, false);
                    const f16x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d0, 1.f, true);
                    const f16x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d1, 1.f, false);
                    const f16x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d1, 1.f, true);
                    wh[i][q] = f16x8{p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
                }
            f16x8 b[2][4];
            auto read_b = [&](int j) {
#pragma unroll
                for (int q = 0; q < 4; q++) b[j & 1][q] = *(const f16x8*)(xs + 16 * j * XB + xo[q]);
            };
            read_b(0);
#pragma unroll
            for (int j = 0; j < MB; j++) {
                if (j + 1 < MB) read_b(j + 1);
                const float f = row_scale(j);
                f32x4 p[RB];
#pragma unroll
                for (int i = 0; i < RB; i++) p[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int q = 0; q < 4; q++)
#pragma unroll
                    for (int i = 0; i < RB; i++) p[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[i][q], b[j & 1][q], p[i], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < RB; i++) {
                    const float g = f * __uint_as_float(sw[GLU && i >= 2 ? 1 : 0]);
#pragma unroll
                    for (int q = 0; q < 4; q++) acc[i][j][q] = __builtin_fmaf(p[i][q], g, acc[i][j][q]);
                }
            }
        } else {
            i32x8 wv[RB], b[2];
#pragma unroll
            for (int i = 0; i < RB; i++) wv[i] = f8_operand(w[i][0], w[i][1]);
            auto read_b = [&](int j) {
                b[j & 1] = f8_operand(*(const u32x4*)(xs + 16 * j * XB + xo[0]), *(const u32x4*)(xs + 16 * j * XB + xo[1]));
            };
            read_b(0);
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
                if (i == 0 && j + 1 < MB) read_b(j + 1);
                if constexpr (KIND == E8S) {
                    acc[i][j] = f8_mfma_at(wv[i], b[j & 1], acc[i][j], sw[0], j < 4 ? sx.x : sx.y, j & 3);
                } else {
                    if (i == 0) f[j & 1] = row_scale(j) * __uint_as_float(sw[0]);
                    p[n % 3] = f8_mfma(wv[i], b[j & 1], f32x4{0.f, 0.f, 0.f, 0.f}, 127u, 127u);
                    if (n >= 2) apply(n - 2);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (KIND == F32S) {
                apply(NP - 2);
                apply(NP - 1);
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
                *(u32x2*)(smem + (16 * j + l16) * 272 + (32 * wave + 16 * i + 4 * c) * 2) = u32x2{o[0], o[1]};
            }
        lds_barrier();
        for (int m = tid >> 4; m < count; m += 64 * G_WAVES / 16) {
            F8Raw<F8BF16, 8> v;
            v.v[0] = *(const u32x4*)(smem + m * 272 + 16 * l16);
            uint32_t top = v.amax();
#pragma unroll
            for (int o = 8; o; o >>= 1) {
                const uint32_t b = (uint32_t)__shfl_xor((int)top, o, 16);
                top = b > top ? b : top;
            }
            uint32_t byte = f8_scale_byte(top);
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
            const int rid = rid_s[16 * j + l16];
            if (rid < 0) continue;
            const bool seen = !a.lhs || xrow(16 * j + l16) >= 0;
#pragma unroll
            for (int i = 0; i < RB; i++) {
                const int64_t n = n0 + 16 * i + 4 * c;
                u32x2 o;
                if (a.half) {
                    o.x = f32_to_f16(acc[i][j][0]) | (uint32_t)f32_to_f16(acc[i][j][1]) << 16;
                    o.y = f32_to_f16(acc[i][j][2]) | (uint32_t)f32_to_f16(acc[i][j][3]) << 16;
                } else {
                    o.x = cvt_pk_bf16(acc[i][j][0], acc[i][j][1]);
                    o.y = cvt_pk_bf16(acc[i][j][2], acc[i][j][3]);
                }
                if (!seen) o = u32x2{0, 0};
                uint16_t* p = y + (int64_t)rid * a.N + n;
                if (wide) {
                    if (n < a.N) *(u32x2*)p = o;
                } else {
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        if (n + q < a.N) p[q] = (uint16_t)(o[q >> 1] >> (16 * (q & 1)));
                }
            }
        }
    }
}

// x's rows into codes [rows, ld] (tails zero) and scale bytes [rows, sld]: 16
// lanes per row and block.  HALF: the codes' values in float16 instead.
template <class T, bool HALF_>
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
    uint32_t top = v.amax();
#pragma unroll
    for (int o = 8; o; o >>= 1) {
        const uint32_t t = (uint32_t)__shfl_xor((int)top, o, 16);
        top = t > top ? t : top;
    }
    // a block with an infinity or a NaN: NaN codes, so the scale stays a number
    uint32_t byte = f8_scale_byte(top);
    const bool nan = byte == 255;
    if (nan) byte = 127;
    const float scale = __uint_as_float(byte << 23);
    const uint32_t c0 = nan ? 0x7f7f7f7fu : v.codes(0, scale), c1 = nan ? 0x7f7f7f7fu : v.codes(1, scale);
    if constexpr (HALF_) {
        u32x4 o;
        o.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c0, 1.f, false));
        o.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c0, 1.f, true));
        o.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c1, 1.f, false));
        o.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c1, 1.f, true));
        *(u32x4*)(q + r * ld + 2 * k) = o;
    } else {
        *(u32x2*)(q + r * ld + k) = u32x2{c0, c1};
    }
    if (l == 0) s[r * sld + b] = (unsigned char)byte;
}

template <int MB, Kind KIND, bool GLU>
int go(const F8Args& a, int64_t tiles, hipStream_t st) {
    if (a.K > FP8_GEMM_MAX_K || a.xld != fp8_row_bytes(a.K, KIND == HALF)) {
        set_error("fp8: K=%lld on tiles", (long long)a.K);
        return EINVAL_ARG;
    }
    const int KB = (int)ceil_div(a.K, F8_BLOCK);
    const int nblocks = (int)ceil_div(a.N, GLU ? 128 : 256);
    const size_t stages = (size_t)G_STAGES * 16 * MB * (KIND == HALF ? 256 : 128) + (size_t)KB * 128;
    const size_t lds = GLU && stages < (size_t)16 * MB * 272 ? (size_t)16 * MB * 272 : stages;
    const int64_t wgs = a.tiles ? ceil_div(tiles, 16) * 16 * nblocks : ceil_div(tiles * nblocks, 8) * 8;
    if (wgs >= (1LL << 31)) {
        set_error("fp8: grid of %lld workgroups", (long long)wgs);
        return EINVAL_ARG;
    }
    allow_dynamic_lds_once((const void*)f8_gemm<MB, KIND, GLU>);
    f8_gemm<MB, KIND, GLU><<<(unsigned)wgs, 64 * G_WAVES, lds, st>>>(a, nblocks, (int)tiles);
    KMI_CHECK_LAUNCH("fp8 tiles");
    return OK;
}

}  // namespace

int64_t fp8_row_bytes(int64_t K, bool half) { return ceil_div(K, F8_BLOCK) * F8_BLOCK * (half ? 2 : 1); }
int64_t fp8_row_scales(int64_t K) { return ceil_div(ceil_div(K, F8_BLOCK), 4) * 4; }

int launch_fp8_rows(const void* x, int dtype, int64_t rows, int64_t K, bool half, unsigned char* q, unsigned char* s,
                    hipStream_t st) {
    const int64_t KB = ceil_div(K, F8_BLOCK), grid = ceil_div(rows * KB, 16);
    if (grid >= (1LL << 31)) {
        set_error("fp8: %lld rows", (long long)rows);
        return EINVAL_ARG;
    }
    const int64_t ld = fp8_row_bytes(K, half), sld = fp8_row_scales(K);
#define KMI_ROWS(T, H) f8_rows<T, H><<<(unsigned)grid, 256, 0, st>>>((const uint16_t*)x, rows, (int)K, (int)KB, q, ld, s, sld)
    if (half) {
        if (dtype == BF16) KMI_ROWS(F8BF16, true);
        else KMI_ROWS(F8F16, true);
    } else {
        if (dtype == BF16) KMI_ROWS(F8BF16, false);
        else KMI_ROWS(F8F16, false);
    }
#undef KMI_ROWS
    KMI_CHECK_LAUNCH("fp8 rows");
    return OK;
}

int launch_fp8_gemm(const F8Args& a, bool glu, int64_t tiles, hipStream_t st) {
    if (glu) return go<4, HALF, true>(a, tiles, st);
    if (a.tm <= 64) return a.e8 ? go<4, E8S, false>(a, tiles, st) : go<4, F32S, false>(a, tiles, st);
    return a.e8 ? go<8, E8S, false>(a, tiles, st) : go<8, F32S, false>(a, tiles, st);
}

}  // namespace kmi
