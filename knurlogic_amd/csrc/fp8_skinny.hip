// Block-scaled E4M3 products of few rows: up to 64 activation rows per tile
// against 16 weight rows (gate|up: 16 gate and the 16 up rows beside them) per
// workgroup.
//
// The 8 waves split K: wave v takes the 128-input blocks v, v + 8, ... and sums
// its own products; the waves' sums are added in LDS, in wave order.  A weight
// row's 128 bytes go from memory into the matrix operand as they are (lane l:
// row l % 16, bytes 16 (l / 16) .. + 15 and the same 64 further, x laid out
// alike), and each wave quantizes the x blocks that it multiplies itself, while
// its weights are on their way: one launch, no pass over x before it.
#include "fp8.hpp"

namespace kmi {

namespace {

constexpr int SK_WAVES = 8;
constexpr int SK_DEPTH = 4;          // weight blocks in flight per wave

template <class T, int MB, bool GLU>
__global__ __launch_bounds__(64 * SK_WAVES) void f8_skinny(F8Args a) {
    constexpr int RB = GLU ? 2 : 1;
    __shared__ __align__(16) float red[SK_WAVES][RB * MB][64][4];
    __shared__ int rid_s[16 * MB], xrow_s[16 * MB];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, c = lane >> 4;
    int64_t expert = 0, start = (int64_t)blockIdx.y * a.tm;
    int count = (int)(a.rows - start < a.tm ? a.rows - start : a.tm);
    if (a.tiles) {
        const int32_t* t = a.tiles + 3 * (int64_t)blockIdx.y;
        expert = t[0]; start = t[1]; count = t[2];
    }
    if (count <= 0) return;                                  // (the whole workgroup)
    const int64_t n0 = (int64_t)blockIdx.x * 16;
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

    const int K = (int)a.K, KB = (K + F8_BLOCK - 1) / F8_BLOCK;
    // the fragments' first rows, and this lane's offset from them (rows past
    // the last repeat it: their sums are not stored)
    const unsigned char* wb[RB];
    int64_t sb[RB];
    uint32_t wo[RB];
    const int64_t SB = (a.wrows + F8_BLOCK - 1) / F8_BLOCK;
#pragma unroll
    for (int i = 0; i < RB; i++) {
        const int64_t r = n0 + (i ? a.N : 0);                // up rows follow the N gate rows
        const int64_t left = (i || !GLU ? a.wrows : a.N) - r;
        wb[i] = a.w + (expert * a.wrows + r) * a.K;
        wo[i] = (uint32_t)(l16 < left ? l16 : (int)left - 1) * (uint32_t)K + 16u * c;
        sb[i] = (expert * SB + r / F8_BLOCK) * KB;
    }
    const typename T::storage* xp[MB];
    bool seen[MB];
#pragma unroll
    for (int i = 0; i < MB; i++) {
        const int xr = xrow_s[16 * i + l16];
        seen[i] = xr >= 0;
        xp[i] = (const typename T::storage*)a.x + (int64_t)(seen[i] ? xr : 0) * a.K;
    }

    auto load_w = [&](int kb, int i) -> i32x8 {
        const int k = kb * F8_BLOCK;
        u32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
        if (k + 16 * c < K) lo = *(const u32x4*)(wb[i] + k + wo[i]);
        if (k + 64 + 16 * c < K) hi = *(const u32x4*)(wb[i] + k + 64 + wo[i]);
        return i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
    };
    f32x4 acc[RB][MB];
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int j = 0; j < MB; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    i32x8 wr[SK_DEPTH][RB];
#pragma unroll
    for (int d = 0; d < SK_DEPTH; d++)
#pragma unroll
        for (int i = 0; i < RB; i++)
            if (wave + SK_WAVES * d < KB) wr[d][i] = load_w(wave + SK_WAVES * d, i);
    for (int kb0 = wave; kb0 < KB; kb0 += SK_WAVES * SK_DEPTH) {
#pragma unroll
        for (int d = 0; d < SK_DEPTH; d++) {
            const int kb = kb0 + SK_WAVES * d;
            if (kb >= KB) break;
            float f[RB];
#pragma unroll
            for (int i = 0; i < RB; i++)
                f[i] = a.e8 ? e8m0_to_f32(((const unsigned char*)a.s)[sb[i] + kb]) : ((const float*)a.s)[sb[i] + kb];
            i32x8 xq[MB];
            float xs[MB];
#pragma unroll
            for (int j = 0; j < MB; j++) {
                F8Raw<T, 16> lo, hi;
                const int k = kb * F8_BLOCK + 16 * c;
                if (k < K) lo.load(xp[j] + k);
                else lo.zero();
                if (k + 64 < K) hi.load(xp[j] + k + 64);
                else hi.zero();
                const uint32_t ma = lo.amax(), mb = hi.amax();
                xs[j] = e8m0_to_f32(f8_scale_byte(f8_max_quads(ma > mb ? ma : mb)));
                const float scale = xs[j];
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    xq[j][q] = (int)lo.codes(q, scale);
                    xq[j][4 + q] = (int)hi.codes(q, scale);
                }
            }
#pragma unroll
            for (int i = 0; i < RB; i++)
#pragma unroll
                for (int j = 0; j < MB; j++) {
                    // codes' products first, then both scales at once: no step
                    // leaves float32's range that the result does not
                    const f32x4 p = f8_mfma(wr[d][i], xq[j], f32x4{0.f, 0.f, 0.f, 0.f}, 127u, 127u);
                    const float g = f[i] * xs[j];
#pragma unroll
                    for (int q = 0; q < 4; q++) acc[i][j][q] = __builtin_fmaf(p[q], g, acc[i][j][q]);
                }
            const int next = kb + SK_WAVES * SK_DEPTH;
            if (next < KB) {
#pragma unroll
                for (int i = 0; i < RB; i++) wr[d][i] = load_w(next, i);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int j = 0; j < MB; j++) *(f32x4*)red[wave][i * MB + j][lane] = acc[i][j];
    __syncthreads();
    // D: row 4 (l / 16) + q of the fragment, token l % 16
    for (int idx = tid; idx < MB * 64; idx += 64 * SK_WAVES) {
        const int j = idx >> 6, l = idx & 63;
        const int tok = 16 * j + (l & 15), rid = rid_s[tok];
        if (rid < 0) continue;
        f32x4 v[RB];
#pragma unroll
        for (int i = 0; i < RB; i++) {
            v[i] = *(const f32x4*)red[0][i * MB + j][l];
#pragma unroll
            for (int w = 1; w < SK_WAVES; w++) {
                const f32x4 o = *(const f32x4*)red[w][i * MB + j][l];
#pragma unroll
                for (int q = 0; q < 4; q++) v[i][q] += o[q];
            }
        }
        typename T::storage* y = (typename T::storage*)a.y + (int64_t)rid * a.N;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int64_t n = n0 + 4 * (l >> 4) + q;
            if (n >= a.N) continue;
            float o = v[0][q];
            if constexpr (GLU) o = silu_bf16r(T::round(v[0][q])) * T::round(v[1][q]);
            y[n] = T::store(xrow_s[tok] >= 0 ? o : 0.f);
        }
    }
}

}  // namespace

int launch_fp8_skinny(const F8Args& a, int dtype, bool glu, int64_t tiles, hipStream_t st) {
    const int64_t nb = ceil_div(a.N, 16);
    if (tiles <= 0 || tiles >= 65536 || nb >= (1LL << 31) || a.tm < 1 || a.tm > 64 || (glu && dtype != BF16)) {
        set_error("fp8: %lld tiles of %d rows", (long long)tiles, a.tm);
        return EINVAL_ARG;
    }
    const dim3 grid((unsigned)nb, (unsigned)tiles);
    const int mb = a.tm <= 16 ? 1 : a.tm <= 32 ? 2 : 4;
#define KMI_SK(T, G)                                                                  \
    do {                                                                              \
        if (mb == 1) f8_skinny<T, 1, G><<<grid, 64 * SK_WAVES, 0, st>>>(a);           \
        else if (mb == 2) f8_skinny<T, 2, G><<<grid, 64 * SK_WAVES, 0, st>>>(a);      \
        else f8_skinny<T, 4, G><<<grid, 64 * SK_WAVES, 0, st>>>(a);                   \
    } while (0)
    if (glu) KMI_SK(F8BF16, true);
    else if (dtype == BF16) KMI_SK(F8BF16, false);
    else KMI_SK(F8F16, false);
#undef KMI_SK
    KMI_CHECK_LAUNCH("fp8 product");
    return OK;
}

}  // namespace kmi
