// E4M3 with one E8M0 scale per block of 128 x 128: weights into codes and
// scales, and back.  Codes from weights are bound by HBM: bf16 [14336, 4096] 30 us, 5.8
// TB/s read and written; a few small experts (5 of [700, 1040], float32) by one
// workgroup's read, maximum and write in sequence, 6.8 us (270 workgroups on 256
// CUs).  The way back is a plain loop whose time nobody waits for at load: 147 us for
// the same bf16 weight, 1.2 TB/s.
#include "fp8.hpp"
#include "../../include/knurlogic_amd.h"

namespace kmi {

namespace {

// One workgroup per block: 16 lanes hold a row of it (8 elements each), 16 rows
// per pass, the whole block in registers between its largest magnitude and its
// codes -- w is read once.
template <class T>
__global__ __launch_bounds__(256) void f8_quantize_blocks(const typename T::storage* __restrict__ w, int64_t rows,
                                                          int64_t cols, int64_t nb, int64_t kb,
                                                          uint32_t* __restrict__ wq, unsigned char* __restrict__ sc) {
    __shared__ uint32_t part[4];
    const int64_t id = blockIdx.x;
    const int64_t k = id % kb, n = id / kb % nb, e = id / (kb * nb);
    const int tid = threadIdx.x, r0 = tid >> 4, c = tid & 15;
    const int64_t col = k * F8_BLOCK + 8 * c, row0 = n * F8_BLOCK + r0;
    const int64_t base = e * rows;
    F8Raw<T, 8> v[8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int64_t r = row0 + 16 * i;
        if (r < rows && col < cols) v[i].load(w + (base + r) * cols + col);
        else v[i].zero();
        const uint32_t b = v[i].amax();
        m = b > m ? b : m;
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        const uint32_t b = (uint32_t)__shfl_xor((int)m, o, 64);
        m = b > m ? b : m;
    }
    if ((tid & 63) == 0) part[tid >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++) m = part[i] > m ? part[i] : m;
    const uint32_t byte = f8_scale_byte(m);
    // a block with an infinity or a NaN: scale NaN, codes 0
    const float scale = __uint_as_float(byte << 23);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int64_t r = row0 + 16 * i;
        if (r >= rows || col >= cols) continue;
        u32x2 o = {v[i].codes(0, scale), v[i].codes(1, scale)};
        if (byte == 255) o = u32x2{0, 0};
        *(u32x2*)(wq + ((base + r) * cols + col) / 4) = o;
    }
    if (tid == 0) sc[id] = (unsigned char)byte;
}

// 16 codes per thread: value = code * scale in float32, rounded to the type
template <class T>
__global__ __launch_bounds__(256) void f8_dequantize(const uint32_t* __restrict__ wq, const void* __restrict__ s,
                                                     int e8, int64_t batch, int64_t rows, int64_t cols, int64_t nb,
                                                     int64_t kb, typename T::storage* __restrict__ out) {
    const int64_t per = cols / 16, n = batch * rows * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per, p = i % per, e = r / rows;
        const int64_t si = (e * nb + r % rows / F8_BLOCK) * kb + p * 16 / F8_BLOCK;
        const float f = e8 ? e8m0_to_f32(((const unsigned char*)s)[si]) : ((const float*)s)[si];
        const u32x4 q = *(const u32x4*)(wq + i * 4);
        typename T::storage* o = out + i * 16;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            o[4 * j + 0] = T::store(__builtin_amdgcn_cvt_f32_fp8((int)q[j], 0) * f);
            o[4 * j + 1] = T::store(__builtin_amdgcn_cvt_f32_fp8((int)q[j], 1) * f);
            o[4 * j + 2] = T::store(__builtin_amdgcn_cvt_f32_fp8((int)q[j], 2) * f);
            o[4 * j + 3] = T::store(__builtin_amdgcn_cvt_f32_fp8((int)q[j], 3) * f);
        }
    }
}

}  // namespace

}  // namespace kmi

using namespace kmi;

extern "C" {

int kmi_quantize_fp8(const void* w, int dtype, int64_t batch, int64_t rows, int64_t cols, uint32_t* wq,
                     uint8_t* scales, void* stream) {
    clear_error();
    KMI_CHECK_ARG(dtype >= BF16 && dtype <= F32, "quantize (fp8): bad dtype %d", dtype);
    KMI_CHECK_ARG(batch >= 0 && rows >= 0 && cols >= 0 && cols % 16 == 0,
                  "quantize (fp8): [%lld, %lld, %lld] (columns in multiples of 16)", (long long)batch,
                  (long long)rows, (long long)cols);
    const int64_t nb = ceil_div(rows, F8_BLOCK), kb = ceil_div(cols, F8_BLOCK), blocks = batch * nb * kb;
    if (blocks == 0) return OK;
    KMI_CHECK_ARG(w && wq && scales, "quantize (fp8): null pointer");
    KMI_CHECK_ARG(((uintptr_t)w | (uintptr_t)wq) % 16 == 0, "quantize (fp8): w and wq on 16 bytes");
    KMI_CHECK_ARG(blocks < (1LL << 31), "quantize (fp8): %lld blocks", (long long)blocks);
    hipStream_t st = (hipStream_t)stream;
    const unsigned g = (unsigned)blocks;
    if (dtype == BF16)
        f8_quantize_blocks<F8BF16><<<g, 256, 0, st>>>((const uint16_t*)w, rows, cols, nb, kb, wq, scales);
    else if (dtype == F16)
        f8_quantize_blocks<F8F16><<<g, 256, 0, st>>>((const uint16_t*)w, rows, cols, nb, kb, wq, scales);
    else
        f8_quantize_blocks<F8F32><<<g, 256, 0, st>>>((const float*)w, rows, cols, nb, kb, wq, scales);
    KMI_CHECK_LAUNCH("quantize (fp8)");
    return OK;
}

int kmi_dequantize_fp8(const uint32_t* wq, const void* scales, int e8m0, int64_t batch, int64_t rows, int64_t cols,
                       void* out, int out_dtype, void* stream) {
    clear_error();
    KMI_CHECK_ARG(out_dtype >= BF16 && out_dtype <= F32, "dequantize (fp8): bad dtype %d", out_dtype);
    KMI_CHECK_ARG(batch >= 0 && rows >= 0 && cols >= 0 && cols % 16 == 0,
                  "dequantize (fp8): [%lld, %lld, %lld] (columns in multiples of 16)", (long long)batch,
                  (long long)rows, (long long)cols);
    const int64_t n = batch * rows * (cols / 16);
    if (n == 0) return OK;
    KMI_CHECK_ARG(wq && scales && out, "dequantize (fp8): null pointer");
    KMI_CHECK_ARG((uintptr_t)wq % 16 == 0, "dequantize (fp8): codes on 16 bytes");
    const int64_t nb = ceil_div(rows, F8_BLOCK), kb = ceil_div(cols, F8_BLOCK), g = ceil_div(n, 256);
    const unsigned grid = (unsigned)(g < (1 << 20) ? g : (1 << 20));
    hipStream_t st = (hipStream_t)stream;
    if (out_dtype == BF16)
        f8_dequantize<F8BF16><<<grid, 256, 0, st>>>(wq, scales, e8m0, batch, rows, cols, nb, kb, (uint16_t*)out);
    else if (out_dtype == F16)
        f8_dequantize<F8F16><<<grid, 256, 0, st>>>(wq, scales, e8m0, batch, rows, cols, nb, kb, (uint16_t*)out);
    else
        f8_dequantize<F8F32><<<grid, 256, 0, st>>>(wq, scales, e8m0, batch, rows, cols, nb, kb, (float*)out);
    KMI_CHECK_LAUNCH("dequantize (fp8)");
    return OK;
}

}  // extern "C"
