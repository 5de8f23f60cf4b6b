// Block-scaled E4M3 products of few rows: tiles of up to 16 activation rows
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
// up rows beside it.  An expert block's products have float16 operands, which hold
// the codes exactly: gate|up's results are rounded to E4M3 again, and the down
// product's to bfloat16 before the combine, where the 8-bit instruction's 1.2e-5
// moved 1 result in 200 to its neighbour (the block's error against float64 0.00170,
// 0.00165 so; 1 token of 128 experts [2048, 768] 20.9 us with either, 4 tokens of top 2
// of 8 [4096, 4096] 76.8 for 73.7).
//
// Bound by x's quantization, which each wave does for its part before its first
// product, and the weights' stream after it (kernel trace, no weights in a cache: 16
// rows of [14336, 4096] 18-19 us, 3.2 TB/s), and where the weights are small by the
// launch and one chain of latencies (1 row of [4096, 4096] 7.0-7.9 us, 2.3 TB/s).
#include "fp8.hpp"

namespace kmi {

namespace {

constexpr int ST_WAVES = 8;
constexpr uint32_t ST_NONE = 0x80000000u;

// the 16 x 16 products' sums of one block, times 2^(sw - 127) 2^(sx - 127)
template <bool EXACT>
__device__ __forceinline__ f32x4 st_times(const i32x8& w, const i32x8& x, uint32_t sw, uint32_t sx) {
    f32x4 p = {0.f, 0.f, 0.f, 0.f};
    if constexpr (EXACT) {
#pragma unroll
        for (int q = 0; q < 4; q++) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(f8_halves(w, q), f8_halves(x, q), p, 0, 0, 0);
        const int e = (int)(sw + sx) - 254;
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = __builtin_amdgcn_ldexpf(p[i], e);
        return p;
    } else {
        return f8_mfma(w, x, p, sw, sx);
    }
}

// workgroups of W waves that run at once on a CU: 3 of 4 waves (GLU), else 2 of 8,
// or 1 where K has 8 parts, with twice the registers (16 rows [8192, 4096]: 14.7 us, 18.1
// with 2; [14336, 4096]: 19.3, 20.7)
template <int KP, int W>
constexpr int st_at_once = W == 4 ? 3 : KP == 8 ? 1 : 2;

// R row blocks per wave and step; KPW blocks of K per wave at most.
// The weights' loads are ordinary ones: non-temporal, [28672, 4096] x 1 row took 28.8 us
// for 26.0, 8 pairs of 64 experts [2048, 2048] 13.0 for 11.6 ([4096, 4096] x 1 row: 7.3 for 7.7).
template <class T, int KP, int KPW, int R, bool GLU, bool EXACT, int W>
__global__ __launch_bounds__(64 * W, (st_at_once<KP, W> * W / 4)) void f8_stream(F8Args a, int steps) {
    constexpr int RB = GLU ? 2 : 1, NP = W / KP, F = R * RB * KPW;
    // weight blocks (2 KB) in flight per wave: 8, or 4 where x, or float16 operands,
    // take the registers
    constexpr int DEPTH = GLU || KPW >= 16 || (EXACT && KP < 8) ? 4 : 8, D = F < DEPTH ? F : DEPTH;
    constexpr int BATCH = KPW < 4 ? KPW : 4;       // x blocks quantized at a time
    static_assert(F % D == 0 && KPW % BATCH == 0, "ring");
    // a wave's x codes, and after them its sums (two steps'), in turn
    constexpr int SUMS = R * RB * 1024, AREA = 2 * SUMS > BATCH * 2048 ? 2 * SUMS : BATCH * 2048;
    __shared__ __align__(16) unsigned char area[W][AREA];
    __shared__ unsigned char xe[W][BATCH * 16];
    __shared__ int rid_s[16], xrow_s[16];
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
    if (a.route) {
        expert = __builtin_amdgcn_readfirstlane(a.route[start]);
        count = 1;
        if (expert < 0 || expert >= a.E) {                   // a zero row (gate|up: not read)
            if (!GLU)
                for (int64_t n = (int64_t)blockIdx.x * blockDim.x + tid; n < a.N; n += (int64_t)gridDim.x * blockDim.x)
                    ((typename T::storage*)a.y)[start * a.N + n] = 0;
            return;
        }
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
            rs, (int)(16 * c < in ? off : ST_NONE), kb * F8_BLOCK, 0));
        const u32x4 hi = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
            rs, (int)(64 + 16 * c < in ? off : ST_NONE), kb * F8_BLOCK + 64, 0));
        wr[q % D] = f8_operand(lo, hi);
    };
    int step = (int)blockIdx.x;
    load_scales(step);
#pragma unroll
    for (int q = 0; q < D; q++) load(q, step);

    if (tid < 16) {
        int rid = -1, xr = -1;
        if (tid < count) {
            rid = a.tiles ? a.sorted[start + tid] : (int)(start + tid);
            xr = rid;
            if (a.tiles || a.route) {
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
    i32x8 x[KPW];
    uint32_t xb[KPW];                                        // the blocks' scale bytes
#pragma unroll
    for (int b0 = 0; b0 < KPW; b0 += BATCH) {
        const int kb = kp + KP * (b0 + c), k = kb * F8_BLOCK + 8 * l16;
        if (kp + KP * b0 >= KB) {                            // (no block of this batch)
#pragma unroll
            for (int i = b0; i < b0 + BATCH; i++) {
                x[i] = i32x8{0, 0, 0, 0, 0, 0, 0, 0};
                xb[i] = 127;
            }
            continue;
        }
        auto rows = [&](int m0, auto many) {                 // several rows' loads before the first is used
            constexpr int G = decltype(many)::value;
            F8Raw<T, 8> v[G];
#pragma unroll
            for (int g = 0; g < G; g++) {
                const int xr = xrow_s[m0 + g < count ? m0 + g : count - 1];
                if (c < BATCH && k < K) v[g].load((const typename T::storage*)a.x + (int64_t)(xr < 0 ? 0 : xr) * a.K + k);
                else v[g].zero();
            }
#pragma unroll
            for (int g = 0; g < G; g++) {
                uint32_t byte = f8_scale_byte(f8_max16(v[g].amax()));
                const bool nan = byte == 255;                // NaN codes, so the scale stays a number
                if (nan) byte = 127;
                const float scale = __uint_as_float(byte << 23);
                const u32x2 o = nan ? u32x2{0x7f7f7f7fu, 0x7f7f7f7fu} : u32x2{v[g].codes(0, scale), v[g].codes(1, scale)};
                const int m = m0 + g;
                if (c < BATCH && m < count) {
                    *(u32x2*)(area[wave] + (c * 16 + m) * 128 + 16 * ((l16 >> 1) ^ (m & 7)) + 8 * (l16 & 1)) = o;
                    if (l16 == 0) xe[wave][c * 16 + m] = (unsigned char)byte;
                }
            }
        };
        if (count == 1) rows(0, std::integral_constant<int, 1>());
        else
            for (int m = 0; m < count; m += 8) rows(m, std::integral_constant<int, 8>());
        // (a wave reads what it wrote: LDS is in order within it)
#pragma unroll
        for (int i = 0; i < BATCH; i++) {
            const int m = l16;
            const bool on = m < count && kp + KP * (b0 + i) < KB;
            const unsigned char* row = area[wave] + (i * 16 + m) * 128;
            i32x8 v = f8_operand(*(const u32x4*)(row + 16 * (c ^ (m & 7))), *(const u32x4*)(row + 16 * ((c + 4) ^ (m & 7))));
#pragma unroll
            for (int q = 0; q < 8; q++) v[q] = on ? v[q] : 0;
            x[b0 + i] = v;
            xb[b0 + i] = on ? xe[wave][i * 16 + m] : 127;
        }
    }

    for (int buf = 0; step < steps; buf ^= 1) {
        const int next = step + (int)gridDim.x;
        // (opaque: float16 operands are made where they are used, not kept)
#pragma unroll
        for (int i = 0; i < KPW; i++) asm volatile("" : "+v"(x[i]));
        uint32_t se[RB];                                     // the step's scales: bytes and mantissas
        float s[RB];
#pragma unroll
        for (int g = 0; g < RB; g++) f8_split(a.e8 ? e8m0_to_f32(sv[g]) : __uint_as_float(sv[g]), se[g], s[g]);
        load_scales(next);
        f32x4 acc[R][RB];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int g = 0; g < RB; g++) acc[r][g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < F; q++) {
            const int g = q % RB, i = q / RB % KPW, r = q / RB / KPW;
            const float sm = __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(s[g]), i));
            const uint32_t sw = (uint32_t)__builtin_amdgcn_readlane((int)se[g], i);
            const f32x4 p = st_times<EXACT>(wr[q % D], x[i], sw, xb[i]);
            const float f = kp + KP * i < KB ? sm : 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++) acc[r][g][e] = __builtin_fmaf(p[e], f, acc[r][g][e]);
            load((q + D) % F, q + D < F ? step : next);
            if constexpr (EXACT) __builtin_amdgcn_sched_barrier(0);    // one block's float16 operands at a time
        }
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int g = 0; g < RB; g++) *(f32x4*)(area[wave] + buf * SUMS + (r * RB + g) * 1024 + 16 * lane) = acc[r][g];
        lds_barrier();
        // D: row 4 (l / 16) + e of the block, activation row l % 16
        for (int idx = tid; idx < NP * R * 64; idx += 64 * W) {
            const int l = idx & 63, r = idx / 64 % R, p = idx / 64 / R;
            const int tok = l & 15, rid = rid_s[tok];
            if (rid < 0) continue;
            f32x4 v[RB];
#pragma unroll
            for (int g = 0; g < RB; g++) {
                const int at = buf * SUMS + (r * RB + g) * 1024 + 16 * l;
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

// The down product and the weighted combine of a token's pairs: one workgroup per
// 16 output columns and token, one wave per pair (in turn past 8), so that no
// product leaves the workgroup before it is summed.  K up to CB_MAX_K.  The last
// blocks, fewer than are in flight, go by a branch each: 6 blocks of 768 inputs as 8
// with two empty ones made the block of 1 token 21.5 us for 20.5.
constexpr int CB_MAX_K = 4096, CB_MAX_SLOTS = 64, CB_DEPTH = 8;

__global__ __launch_bounds__(64 * ST_WAVES) void f8_combine(F8Args a, const uint16_t* __restrict__ scores, int k,
                                                            uint16_t* __restrict__ out) {
    __shared__ __align__(16) unsigned char xs[ST_WAVES][CB_MAX_K];
    __shared__ unsigned char xe[ST_WAVES][CB_MAX_K / F8_BLOCK];
    __shared__ __align__(16) float sums[CB_MAX_SLOTS][16];
    __shared__ float weight[CB_MAX_SLOTS];
    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, c = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int K = (int)a.K, KB = (K + F8_BLOCK - 1) / F8_BLOCK;
    const int64_t SB = (a.wrows + F8_BLOCK - 1) / F8_BLOCK, n0 = (int64_t)blockIdx.x * 16;
    const int64_t left = a.N - n0 < 16 ? a.N - n0 : 16;
    const int64_t token = blockIdx.y;
    if (tid < k) weight[tid] = bf16_to_f32(scores[token * k + tid]);
    for (int slot = wave; slot < k; slot += ST_WAVES) {
        const int64_t pair = token * k + slot;
        const int64_t expert = __builtin_amdgcn_readfirstlane(a.route[pair]);
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        if (expert >= 0 && expert < a.E) {
            const __amdgpu_buffer_rsrc_t rs = make_rsrc(a.w + (expert * a.wrows + n0) * a.K, left * a.K);
            const uint32_t off = (uint32_t)l16 * (uint32_t)K + 16u * c;
            const int64_t si = (expert * SB + n0 / F8_BLOCK) * KB + (lane < KB ? lane : 0);
            uint32_t sw;
            float sm;
            f8_split(a.e8 ? e8m0_to_f32(((const unsigned char*)a.s)[si]) : ((const float*)a.s)[si], sw, sm);
            i32x8 w[CB_DEPTH];
            auto load = [&](int kb, int d) {
                const int in = K - kb * F8_BLOCK;
                w[d] = f8_operand(
                    __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                        rs, (int)(16 * c < in ? off : ST_NONE), kb * F8_BLOCK, 0)),
                    __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                        rs, (int)(64 + 16 * c < in ? off : ST_NONE), kb * F8_BLOCK + 64, 0)));
            };
#pragma unroll
            for (int d = 0; d < CB_DEPTH; d++) load(d, d);
            // the pair's activations: 16 lanes per block
            for (int b0 = 0; b0 < KB; b0 += 4) {
                const int kk = (b0 + c) * F8_BLOCK + 8 * l16;
                F8Raw<F8BF16, 8> v;
                if (kk < K) v.load((const uint16_t*)a.x + pair * a.K + kk);
                else v.zero();
                uint32_t byte = f8_scale_byte(f8_max16(v.amax()));
                const bool nan = byte == 255;
                if (nan) byte = 127;
                const float scale = __uint_as_float(byte << 23);
                if (b0 + c < KB) {
                    *(u32x2*)(xs[wave] + kk) = nan ? u32x2{0x7f7f7f7fu, 0x7f7f7f7fu} : u32x2{v.codes(0, scale), v.codes(1, scale)};
                    if (l16 == 0) xe[wave][b0 + c] = (unsigned char)byte;
                }
            }
            auto block = [&](int kb, int d) {
                // every column the same row: column 0 is used
                const i32x8 x = f8_operand(*(const u32x4*)(xs[wave] + kb * F8_BLOCK + 16 * c),
                                           *(const u32x4*)(xs[wave] + kb * F8_BLOCK + 64 + 16 * c));
                const f32x4 p = st_times<true>(w[d], x, (uint32_t)__builtin_amdgcn_readlane((int)sw, kb), xe[wave][kb]);
                const float s = __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(sm), kb));
#pragma unroll
                for (int e = 0; e < 4; e++) acc[e] = __builtin_fmaf(p[e], s, acc[e]);
            };
            int b0 = 0;
            for (; b0 + CB_DEPTH <= KB; b0 += CB_DEPTH) {
#pragma unroll
                for (int d = 0; d < CB_DEPTH; d++) {
                    block(b0 + d, d);
                    load(b0 + d + CB_DEPTH, d);
                }
            }
#pragma unroll
            for (int d = 0; d < CB_DEPTH; d++) {             // (few: a branch costs less than an empty block)
                if (b0 + d >= KB) break;
                block(b0 + d, d);
            }
        }
        if (l16 == 0) *(f32x4*)&sums[slot][4 * c] = acc;
    }
    __syncthreads();
    if (tid < left) {
        double o = 0.0;
        for (int s = 0; s < k; s++)
            o += (double)TBF16::round(TBF16::round(sums[s][tid]) * weight[s]);
        float f = (float)o;
        asm volatile("" : "+v"(f));              // rounded to float32 and then to bf16, as moe_combine
        out[token * a.N + n0 + tid] = f32_to_bf16(f);
    }
}

template <class T, int KP, int KPW, int R, bool GLU, bool EXACT, int W = ST_WAVES>
int go(const F8Args& a, int64_t tiles, hipStream_t st) {
    const int64_t steps = ceil_div(a.N, 16 * R * (W / KP));
    if (steps >= (1LL << 31)) {
        set_error("fp8: N=%lld", (long long)a.N);
        return EINVAL_ARG;
    }
    // as many workgroups per tile as keep every one's steps alike and run at once
    // (16 more than that are a second round: 24 pairs [2048, 4096], 528 workgroups
    // 52.1 us, 456 43.1); of sorted tiles some are empty, and a few more run
    // (512 rows of 128 experts [1536, 4096]: 148 us, 181 with the first rule)
    constexpr int64_t most = 256 * st_at_once<KP, W>;
    int64_t per = ceil_div(steps, tiles < most ? most / tiles : 1);
    if (a.tiles) per = ceil_div(steps * tiles, most) < steps ? ceil_div(steps * tiles, most) : steps;
    const int64_t gx = ceil_div(steps, per);
    f8_stream<T, KP, KPW, R, GLU, EXACT, W><<<dim3((unsigned)gx, (unsigned)tiles), 64 * W, 0, st>>>(a, (int)steps);
    KMI_CHECK_LAUNCH("fp8 stream");
    return OK;
}

// The parts of K: as few as leave a wave's x in its registers (KPW blocks), so that
// a part with no block is rare.
template <class T, bool GLU, bool EXACT>
int parts(const F8Args& a, int64_t tiles, hipStream_t st) {
    const int64_t KB = ceil_div(a.K, F8_BLOCK);
    if constexpr (GLU) {
        if (KB <= 4) return go<T, 2, 2, 1, GLU, EXACT, 4>(a, tiles, st);
        if (KB <= 8) return go<T, 2, 4, 1, GLU, EXACT, 4>(a, tiles, st);
        if (KB <= 16) return go<T, 4, 4, 1, GLU, EXACT, 4>(a, tiles, st);
        if (KB <= 32) return go<T, 8, 4, 1, GLU, EXACT>(a, tiles, st);
        if (KB <= 64) return go<T, 8, 8, 1, GLU, EXACT>(a, tiles, st);
    } else {
        if (KB <= 2) return go<T, 2, 1, 4, GLU, EXACT>(a, tiles, st);
        if (KB <= 4) return go<T, 2, 2, 2, GLU, EXACT>(a, tiles, st);
        if (KB <= 8) return go<T, 2, 4, 1, GLU, EXACT>(a, tiles, st);
        if (KB <= 16) return go<T, 4, 4, 1, GLU, EXACT>(a, tiles, st);
        if (KB <= 32) return go<T, 8, 4, 1, GLU, EXACT>(a, tiles, st);
        if (KB <= 64) return go<T, 8, 8, 1, GLU, EXACT>(a, tiles, st);
    }
    if constexpr (!EXACT) return go<T, 8, 16, 1, GLU, EXACT>(a, tiles, st);
    set_error("fp8: K=%lld for tiles of %d rows", (long long)a.K, a.tm);
    return EINVAL_ARG;
}

}  // namespace

int64_t fp8_skinny_max_k(bool block) { return block ? 8192 : 16384; }

int launch_fp8_skinny(const F8Args& a, int dtype, F8Use use, int64_t tiles, hipStream_t st) {
    const bool block = use != F8_PRODUCT;
    if (tiles <= 0 || tiles >= 65536 || a.tm < 1 || a.tm > 16 || (block && dtype != BF16) || a.K > fp8_skinny_max_k(block)) {
        set_error("fp8: %lld tiles of %d rows, K=%lld", (long long)tiles, a.tm, (long long)a.K);
        return EINVAL_ARG;
    }
    if (block) return use == F8_GLU ? parts<F8BF16, true, true>(a, tiles, st) : parts<F8BF16, false, true>(a, tiles, st);
    return dtype == BF16 ? parts<F8BF16, false, false>(a, tiles, st) : parts<F8F16, false, false>(a, tiles, st);
}

bool fp8_combine_supported(int64_t K, int k) { return K <= CB_MAX_K && k <= CB_MAX_SLOTS; }

int launch_fp8_combine(const F8Args& a, const void* scores, int k, int64_t T, void* out, hipStream_t st) {
    const int64_t nb = ceil_div(a.N, 16);
    if (!a.route || !fp8_combine_supported(a.K, k) || T < 1 || T >= 65536 || nb >= (1LL << 31)) {
        set_error("fp8: combine of %lld tokens, K=%lld", (long long)T, (long long)a.K);
        return EINVAL_ARG;
    }
    f8_combine<<<dim3((unsigned)nb, (unsigned)T), 64 * ST_WAVES, 0, st>>>(a, (const uint16_t*)scores, k, (uint16_t*)out);
    KMI_CHECK_LAUNCH("fp8 combine");
    return OK;
}

}  // namespace kmi
