// Block-scaled E4M3 products of few rows: tiles of up to 16 or 32 activation rows
// against 16-row blocks of weights.
//
// The 8 waves of a workgroup split into KP parts of K (part v takes the 128-input
// blocks v, v + KP, ...) and 8 / KP groups of weight rows.  Each wave quantizes the
// x blocks of its part once, into the matrix operand's registers, and streams the
// weights of its share of the row blocks past them, D blocks in flight; a weight
// row's 128 bytes go from memory into the operand as they are (lane l: row l % 16,
// bytes 16 (l / 16) .. + 15 and the same 64 further, x laid out alike).  The parts'
// sums are added in LDS, in order, and one launch does it all: no pass over x
// before, no partial sums in memory.  gate|up takes a block of gate rows and the
// up rows beside it, in float16 operands (its results are rounded to E4M3 again).
#include "fp8.hpp"

namespace kmi {

namespace {

constexpr int ST_WAVES = 8;
constexpr uint32_t ST_NONE = 0x80000000u;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f16x8 st_halves(const i32x8& v, int q) {      // codes 8 q .. 8 q + 7
    const uint32_t d0 = (uint32_t)v[2 * q], d1 = (uint32_t)v[2 * q + 1];
    const f16x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d0, 1.f, false);
    const f16x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d0, 1.f, true);
    const f16x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d1, 1.f, false);
    const f16x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d1, 1.f, true);
    return f16x8{p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
}

// the 16 x 16 products' sums of one block
template <bool HALF>
__device__ __forceinline__ f32x4 st_times(const i32x8& w, const i32x8& x) {
    f32x4 p = {0.f, 0.f, 0.f, 0.f};
    if constexpr (HALF) {
#pragma unroll
        for (int q = 0; q < 4; q++) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(st_halves(w, q), st_halves(x, q), p, 0, 0, 0);
        return p;
    } else {
        return f8_mfma(w, x, p, 127u, 127u);
    }
}

// R row blocks per wave and step; KPW blocks of K per wave at most
template <class T, int MB, int KP, int KPW, int R, bool GLU>
__global__ __launch_bounds__(64 * ST_WAVES) void f8_stream(F8Args a, int steps) {
    constexpr int RB = GLU ? 2 : 1, NP = ST_WAVES / KP, F = R * RB * KPW;
    // weight blocks (2 KB) in flight per wave: 8, or 4 where x takes 128 registers
    constexpr int DEPTH = KPW * MB >= 16 ? 4 : 8, D = F < DEPTH ? F : DEPTH;
    constexpr int BATCH = KPW * MB < 4 ? KPW : 4 / MB;       // x blocks quantized at a time
    static_assert(F % D == 0 && KPW % BATCH == 0, "ring");
    // a wave's x codes, and after them its sums (two steps'), in turn
    constexpr int SUMS = R * RB * MB * 1024, AREA = 2 * SUMS > BATCH * MB * 2048 ? 2 * SUMS : BATCH * MB * 2048;
    __shared__ __align__(16) unsigned char area[ST_WAVES][AREA];
    __shared__ unsigned char xe[ST_WAVES][BATCH * MB * 16];
    __shared__ int rid_s[16 * MB], xrow_s[16 * MB];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kp = wave % KP, np = wave / KP;
    const int l16 = lane & 15, c = lane >> 4;
    int64_t expert = 0, start = (int64_t)blockIdx.y * a.tm;
    int count = (int)(a.rows - start < a.tm ? a.rows - start : a.tm);
    if (a.tiles) {
        const int32_t* t = a.tiles + 3 * (int64_t)blockIdx.y;
        expert = __builtin_amdgcn_readfirstlane(t[0]);
        start = __builtin_amdgcn_readfirstlane(t[1]);
        count = __builtin_amdgcn_readfirstlane(t[2]);
    }
    if (count <= 0) return;                                  // (the whole workgroup)

    // the weights first: they are what the rest waits for
    const int K = (int)a.K, KB = (K + F8_BLOCK - 1) / F8_BLOCK;
    const int64_t SB = (a.wrows + F8_BLOCK - 1) / F8_BLOCK;
    i32x8 wr[D];
    uint32_t sv[RB];                                         // a step's scales, lane i: of K block i
    auto load_scales = [&](int step) {
        const int64_t n = ((int64_t)step * NP + np) * 16 * R;
        const int kb = kp + KP * (lane < KPW ? lane : 0);
#pragma unroll
        for (int g = 0; g < RB; g++) {
            const int64_t row = (step < steps && n < a.N ? n : 0) + (g ? a.N : 0);
            const int64_t i = (expert * SB + row / F8_BLOCK) * KB + (kb < KB ? kb : 0);
            sv[g] = a.e8 ? ((const unsigned char*)a.s)[i] : ((const uint32_t*)a.s)[i];
        }
    };
    auto load = [&](int q, int step) {                       // block q of the step: row block, K block, gate / up
        const int g = q % RB, i = q / RB % KPW, r = q / RB / KPW;
        const int64_t n = ((int64_t)step * NP + np) * 16 * R + 16 * r;
        const int64_t left = step < steps && n < a.N ? (a.N - n < 16 ? a.N - n : 16) : 0;
        const int64_t row = (left ? n : 0) + (g ? a.N : 0);
        const int kb = kp + KP * i;
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(a.w + (expert * a.wrows + row) * a.K, left * a.K);
        // inputs of this block; opaque, or the compiler keeps every block's masks
        // and offsets in registers across the steps
        int in = K - kb * F8_BLOCK;
        asm volatile("" : "+s"(in));
        const uint32_t off = (uint32_t)l16 * (uint32_t)K + 16u * c;
        const u32x4 lo = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
            rs, (int)(16 * c < in ? off : ST_NONE), kb * F8_BLOCK, AUX_NT));
        const u32x4 hi = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
            rs, (int)(64 + 16 * c < in ? off : ST_NONE), kb * F8_BLOCK + 64, AUX_NT));
        wr[q % D] = f8_operand(lo, hi);
    };
    int step = (int)blockIdx.x;
    load_scales(step);
#pragma unroll
    for (int q = 0; q < D; q++) load(q, step);

    if (tid < 16 * MB) {
        int rid = -1, xr = -1;
        if (tid < count) {
            rid = a.tiles ? a.sorted[start + tid] : (int)(start + tid);
            xr = rid;
            if (a.tiles) {
                const int p = rid / (int)a.Mper, m = rid % (int)a.Mper;
                const int64_t b = a.lhs ? a.lhs[p] : p / (int)a.lhs_div;
                const int64_t r = b * a.Mper + m;
                xr = b >= 0 && r < a.xrows ? (int)r : -1;
            }
        }
        rid_s[tid] = rid;
        xrow_s[tid] = xr;
    }
    __syncthreads();

    // x blocks of this part: 16 lanes quantize 128 inputs of a row, BATCH blocks of
    // a row at once, through LDS (pieces permuted by the row) into the operand
    i32x8 x[KPW][MB];
    float xf[KPW][MB];
#pragma unroll
    for (int b0 = 0; b0 < KPW; b0 += BATCH) {
        const int kb = kp + KP * (b0 + c), k = kb * F8_BLOCK + 8 * l16;
        if (kp + KP * b0 >= KB) {                            // (no block of this batch)
#pragma unroll
            for (int i = b0; i < b0 + BATCH; i++)
#pragma unroll
                for (int j = 0; j < MB; j++) {
                    x[i][j] = i32x8{0, 0, 0, 0, 0, 0, 0, 0};
                    xf[i][j] = 0.f;
                }
            continue;
        }
#pragma unroll 4
        for (int m = 0; m < count; m++) {
            const int xr = xrow_s[m];
            F8Raw<T, 8> v;
            if (c < BATCH && k < K) v.load((const typename T::storage*)a.x + (int64_t)(xr < 0 ? 0 : xr) * a.K + k);
            else v.zero();
            uint32_t top = v.amax();
#pragma unroll
            for (int o = 8; o; o >>= 1) {
                const uint32_t u = (uint32_t)__shfl_xor((int)top, o, 16);
                top = u > top ? u : top;
            }
            uint32_t byte = f8_scale_byte(top);
            const bool nan = byte == 255;                    // NaN codes, so the scale stays a number
            if (nan) byte = 127;
            const float scale = __uint_as_float(byte << 23);
            const u32x2 o = nan ? u32x2{0x7f7f7f7fu, 0x7f7f7f7fu} : u32x2{v.codes(0, scale), v.codes(1, scale)};
            if (c < BATCH) {
                *(u32x2*)(area[wave] + (c * MB * 16 + m) * 128 + 16 * ((l16 >> 1) ^ (m & 7)) + 8 * (l16 & 1)) = o;
                if (l16 == 0) xe[wave][c * MB * 16 + m] = (unsigned char)byte;
            }
        }
        // (a wave reads what it wrote: LDS is in order within it)
#pragma unroll
        for (int i = 0; i < BATCH; i++)
#pragma unroll
            for (int j = 0; j < MB; j++) {
                const int m = 16 * j + l16;
                const bool on = m < count && kp + KP * (b0 + i) < KB;
                const unsigned char* row = area[wave] + (i * MB * 16 + m) * 128;
                i32x8 v = f8_operand(*(const u32x4*)(row + 16 * (c ^ (m & 7))), *(const u32x4*)(row + 16 * ((c + 4) ^ (m & 7))));
#pragma unroll
                for (int q = 0; q < 8; q++) v[q] = on ? v[q] : 0;
                x[b0 + i][j] = v;
                xf[b0 + i][j] = on ? __uint_as_float((uint32_t)xe[wave][i * MB * 16 + m] << 23) : 0.f;
            }
    }

    for (int buf = 0; step < steps; buf ^= 1) {
        const int next = step + (int)gridDim.x;
        // (opaque: float16 operands are made where they are used, not kept)
#pragma unroll
        for (int i = 0; i < KPW; i++)
#pragma unroll
            for (int j = 0; j < MB; j++) asm volatile("" : "+v"(x[i][j]));
        float s[RB];
#pragma unroll
        for (int g = 0; g < RB; g++) s[g] = a.e8 ? e8m0_to_f32(sv[g]) : __uint_as_float(sv[g]);
        load_scales(next);
        f32x4 acc[R][RB][MB];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int g = 0; g < RB; g++)
#pragma unroll
                for (int j = 0; j < MB; j++) acc[r][g][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < F; q++) {
            const int g = q % RB, i = q / RB % KPW, r = q / RB / KPW;
            const float sw = __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(s[g]), i));
#pragma unroll
            for (int j = 0; j < MB; j++) {
                // codes' products first, then both scales at once: no step leaves
                // float32's range that the result does not
                const f32x4 p = st_times<GLU>(wr[q % D], x[i][j]);
                const float f = kp + KP * i < KB ? sw * xf[i][j] : 0.f;
#pragma unroll
                for (int e = 0; e < 4; e++) acc[r][g][j][e] = __builtin_fmaf(p[e], f, acc[r][g][j][e]);
            }
            load((q + D) % F, q + D < F ? step : next);
        }
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int g = 0; g < RB; g++)
#pragma unroll
                for (int j = 0; j < MB; j++) *(f32x4*)(area[wave] + buf * SUMS + ((r * RB + g) * MB + j) * 1024 + 16 * lane) = acc[r][g][j];
        lds_barrier();
        // D: row 4 (l / 16) + e of the block, activation row l % 16
        for (int idx = tid; idx < NP * R * MB * 64; idx += 64 * ST_WAVES) {
            const int l = idx & 63, j = idx / 64 % MB, r = idx / 64 / MB % R, p = idx / 64 / MB / R;
            const int tok = 16 * j + (l & 15), rid = rid_s[tok];
            if (rid < 0) continue;
            f32x4 v[RB];
#pragma unroll
            for (int g = 0; g < RB; g++) {
                const int at = buf * SUMS + ((r * RB + g) * MB + j) * 1024 + 16 * l;
                v[g] = *(const f32x4*)(area[p * KP] + at);
#pragma unroll
                for (int w = 1; w < KP; w++) {
                    const f32x4 o = *(const f32x4*)(area[p * KP + w] + at);
#pragma unroll
                    for (int e = 0; e < 4; e++) v[g][e] += o[e];
                }
            }
            typename T::storage* y = (typename T::storage*)a.y + (int64_t)rid * a.N;
            const int64_t n = (((int64_t)step * NP + p) * R + r) * 16 + 4 * (l >> 4);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (n + e >= a.N) continue;
                float o = v[0][e];
                if constexpr (GLU) o = silu_bf16r(T::round(v[0][e])) * T::round(v[1][e]);
                y[n + e] = T::store(xrow_s[tok] >= 0 ? o : 0.f);
            }
        }
        step = next;
    }
}

// waves of the device's CUs that stream at once: two workgroups each
constexpr int64_t ST_GRID = 512;

template <class T, int MB, int KP, int KPW, int R, bool GLU>
int go(const F8Args& a, int64_t tiles, hipStream_t st) {
    const int64_t steps = ceil_div(a.N, 16 * R * (ST_WAVES / KP));
    if (steps >= (1LL << 31)) {
        set_error("fp8: N=%lld", (long long)a.N);
        return EINVAL_ARG;
    }
    // as many workgroups per tile as keep every one's steps alike
    const int64_t per = ceil_div(steps * tiles, ST_GRID);
    const int64_t gx = ceil_div(steps, per < steps ? per : steps);
    f8_stream<T, MB, KP, KPW, R, GLU><<<dim3((unsigned)gx, (unsigned)tiles), 64 * ST_WAVES, 0, st>>>(a, (int)steps);
    KMI_CHECK_LAUNCH("fp8 stream");
    return OK;
}

// The parts of K: 8 where each then has at most KPW blocks, or fewer for a short K
// (a part with no block would idle).
template <class T, int MB, bool GLU>
int parts(const F8Args& a, int64_t tiles, hipStream_t st) {
    const int64_t KB = ceil_div(a.K, F8_BLOCK);
    if (KB <= 2) return go<T, MB, 2, 1, GLU ? 2 : 4, GLU>(a, tiles, st);
    if (KB <= 4) return go<T, MB, 2, 2, GLU ? 1 : 2, GLU>(a, tiles, st);
    if (KB <= 8) return go<T, MB, 2, 4, 1, GLU>(a, tiles, st);
    if (KB <= 16) return go<T, MB, 4, 4, 1, GLU>(a, tiles, st);
    if (KB <= 32) return go<T, MB, 8, 4, 1, GLU>(a, tiles, st);
    if (KB <= 64) return go<T, MB, 8, 8, 1, GLU>(a, tiles, st);
    if constexpr (MB == 1 && !GLU) return go<T, MB, 8, 16, 1, GLU>(a, tiles, st);
    set_error("fp8: K=%lld for tiles of %d rows", (long long)a.K, a.tm);
    return EINVAL_ARG;
}

}  // namespace

int64_t fp8_skinny_max_k(int tm, bool glu) { return tm <= 16 && !glu ? 16384 : 8192; }

int launch_fp8_skinny(const F8Args& a, int dtype, bool glu, int64_t tiles, hipStream_t st) {
    if (tiles <= 0 || tiles >= 65536 || a.tm < 1 || a.tm > (glu ? 16 : 32) || (glu && dtype != BF16) ||
        a.K > fp8_skinny_max_k(a.tm, glu)) {
        set_error("fp8: %lld tiles of %d rows, K=%lld", (long long)tiles, a.tm, (long long)a.K);
        return EINVAL_ARG;
    }
    if (glu) return parts<F8BF16, 1, true>(a, tiles, st);
    if (a.tm <= 16) return dtype == BF16 ? parts<F8BF16, 1, false>(a, tiles, st) : parts<F8F16, 1, false>(a, tiles, st);
    return dtype == BF16 ? parts<F8BF16, 2, false>(a, tiles, st) : parts<F8F16, 2, false>(a, tiles, st);
}

}  // namespace kmi
