// The C entries of the block-scaled E4M3 products: a dense projection, rows
// against their own expert (mlx's gather_qmm), and an expert block's SwitchGLU
// with the weighted combine.
#include "fp8.hpp"
#include "qgemv.hpp"
#include "../../include/knurlogic_amd.h"

namespace kmi {

namespace {

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

constexpr int64_t MAX_E = 4096;        // of the GPU sort

int check_operands(const char* what, int dtype, int64_t K, int64_t N, const void* x, const void* w) {
    KMI_CHECK_ARG(dtype == BF16 || dtype == F16, "%s: dtype %d (bfloat16 or float16)", what, dtype);
    KMI_CHECK_ARG(K > 0 && K % 16 == 0 && K <= FP8_GEMM_MAX_K, "%s: K=%lld (a multiple of 16 up to %lld)", what,
                  (long long)K, (long long)FP8_GEMM_MAX_K);
    KMI_CHECK_ARG(N > 0 && N < (1LL << 31), "%s: N=%lld", what, (long long)N);
    KMI_CHECK_ARG((((uintptr_t)x | (uintptr_t)w) & 15) == 0, "%s: x and w on 16 bytes", what);
    return OK;
}

int check_workspace(const char* what, size_t need, const void* ws, size_t bytes) {
    if (need && (!ws || bytes < need)) {
        set_error("%s: workspace of %zu bytes needed, %zu given", what, need, bytes);
        return EWORKSPACE;
    }
    KMI_CHECK_ARG(((uintptr_t)ws & 15) == 0, "%s: workspace on 16 bytes", what);
    return OK;
}

// How a call runs: on f8_stream, which quantizes x itself, or with x quantized
// ahead on f8_gemm's tiles; and the rows per tile.
struct Plan {
    bool gemm;
    int tm;
    bool pairs;        // f8_stream pair by pair, without the sort
};

//
// (Times at the rules: us per call in a captured graph over 600 MB of different
// weights, so that none is in a cache.)
//
// Dense: the stream up to 16 rows, while each wave's part of x, which it quantizes
// before its first product, is short: 9 rows or more up to K = 4096, 2 or more up to 9216,
// one up to the most.  Stream and tiles at 16 rows: [4096, 4096] 11.6, 14.4;
// [14336, 4096] 19.1, 20.6; [4096, 4352] 15.2, 15.3; [4096, 5120] 17.1, 15.6; [4096,
// 8192] 19.2, 17.4; [4096, 14336] 31.9, 21.4; at 8: [4096, 8192] 15.2, 17.1; [4096, 9216]
// 17.8, 17.8; [14336, 10240] 39.6, 36.6; [4096, 14336] 23.3, 21.0; at 2 the same within 1; at 1:
// [4096, 8192] 11.8, 16.5; [4096, 14336] 17.3, 20.5; [8192, 16384] 32.8, 42.2; but [5120,
// 12288] 23.4, 20.9.  Then the tiles with the least rounds x time of a round.  A block of 128 inputs takes 0.5 us in tiles of 64 rows where each is
// alone on its CU, 0.8 two to a CU; 0.9 and 1.2 in tiles of 128; 1.5 in tiles of 256
// x 256, one to a CU.  [4096, 4096], tiles of 64 / 128 / 256: 512 rows 23 / 35 / 59
// us, 1024 35 / 38 / 60, 2048 63 / 50 / 65, 4096 117 / 94 / 75; [14336, 4096]: 256
// rows 37 / 38 / 62, 512 64 / 49 / 64, 1024 106 / 90 / 67.
Plan plan_dense(int64_t M, int64_t K, int64_t N) {
    if (M <= 16 && K <= (M == 1 ? fp8_skinny_max_k(false) : M <= 8 ? 9216 : 4096)) return {false, 16};
    const auto rounds = [&](int64_t tm, int64_t tn, int64_t at_once) {
        return ceil_div(ceil_div(M, tm) * ceil_div(N, tn), at_once);
    };
    const int64_t t64 = rounds(64, 128, 256) == 1 ? 5 : 8 * rounds(64, 128, 512);
    const int64_t t128 = rounds(128, 128, 256) == 1 ? 9 : 12 * rounds(128, 128, 512);
    const int64_t t256 = 15 * rounds(256, 256, 256);
    return {true, t64 <= t128 && t64 <= t256 ? 64 : t128 <= t256 ? 128 : 256};
}

// Grouped.  Pair by pair (no sort, no tile list; an expert's weights once per pair)
// while few pairs share an expert: 64 experts [2048, 2048], 16 pairs 15.7 us,
// streamed by the sorted list 24.5, tiles 22.5; 32: 25.3, 34.6, 31.7; 64: 42.5,
// 50.5, 47.0; 96: 61.5, 51.1, 48.6; 8 experts [4096, 4096], 8 pairs 22.1, 29.7, 35.1,
// 12: 35.7, 33.4, 43.6.  Then the stream while the tiles would be few (8 experts
// [4096, 4096], 64 rows: 42.8, tiles 45.5, 128 rows 51.3, 48.8; but 64 experts
// [2048, 2048], 256 rows: 61.9, 58.8), or an expert's few rows are long (128 experts
// [1536, 4096], 256 rows: 126, 156, 512 rows: 148, 184; 768: 186, 174; 256 experts
// [2048, 4096], 256 rows, one each: 287, 253).  Tiles of 64 rows (gate|up's only
// size) up to 64 rows to an expert, then 128, as below.  Where the rule takes not the
// best of the three: 128 experts [1536, 4096], 96 rows tiles 109 (stream 84), 128 rows
// tiles 128 (pairs 112); 256 experts [2048, 4096], 96 rows pairs 147 (stream 121); 64
// experts [2048, 2048], 48 rows tiles 40.5 (pairs 36.1); blocks of 32 experts 2048 -> 768, top
// 4, 6 and 8 tokens: stream 37.4 and 41.6 (pairs 33.9 and 37.3): it counts rows to an
// expert, not the bytes each way reads.  Tiles of 64 and 128: 64 experts [2048, 2048], 96 rows each:
// 97 us, in tiles of 64 104; 8 experts [4096, 4096], 64 rows each: 54 both.
Plan plan_grouped(int64_t rows, int64_t P, int64_t E, int64_t K, int64_t N, bool glu) {
    const int64_t experts = P < E ? P : E, per = ceil_div(rows, experts);
    if (K <= fp8_skinny_max_k(glu)) {
        if (rows == P && (2 * P <= E || P <= (E < 8 ? E : 8))) return {false, 16, true};
        if (per <= 8 && experts * ceil_div(N, 128) <= 512) return {false, 16};
        if (2 <= per && per <= 4 && K > 2048) return {false, 16};
    }
    return {true, glu || per <= 64 ? 64 : 128};
}

size_t values_bytes(int64_t rows, int64_t K) { return align256((size_t)rows * fp8_row_bytes(K) * 2); }

// (a part of K may read 16 scale bytes from any word of a row)
size_t rows_bytes(int64_t rows, int64_t K) {
    return align256((size_t)rows * fp8_row_bytes(K)) + align256((size_t)rows * fp8_row_scales(K) + 16);
}

// x quantized at ws (rows_bytes), as a's x
int quantize_rows(F8Args& a, const void* x, int dtype, int64_t rows, char* ws, hipStream_t st) {
    unsigned char* q = (unsigned char*)ws;
    unsigned char* s = q + align256((size_t)rows * fp8_row_bytes(a.K));
    a.x = q; a.xrows = rows; a.xld = fp8_row_bytes(a.K); a.xs = s; a.xs_ld = fp8_row_scales(a.K);
    return launch_fp8_rows(x, dtype, rows, a.K, q, s, st);
}

}  // namespace

}  // namespace kmi

using namespace kmi;

extern "C" {

size_t kmi_qmm_fp8_workspace_bytes(int64_t M, int64_t K, int64_t N, int dtype) {
    if (M <= 0 || K <= 0 || N <= 0) return 0;
    const Plan p = plan_dense(M, K, N);
    if (!p.gemm) return 0;
    const int parts = fp8_gemm_parts(M, K, N, p.tm);
    return rows_bytes(M, K) + (parts > 1 ? (size_t)parts * M * ceil_div(N, 4) * 16 : 0);
}

int kmi_qmm_fp8(const void* x, int64_t M, int64_t K, int64_t N, const uint32_t* w, const void* scales, int e8m0,
                int dtype, void* y, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    const char* what = "qmm (fp8)";
    int rc = check_operands(what, dtype, K, N, x, w);
    if (rc) return rc;
    KMI_CHECK_ARG(M >= 0 && M < (1 << 21), "%s: M=%lld", what, (long long)M);
    if (M == 0) return OK;
    KMI_CHECK_ARG(x && w && scales && y, "%s: null pointer", what);
    rc = check_workspace(what, kmi_qmm_fp8_workspace_bytes(M, K, N, dtype), workspace, workspace_bytes);
    if (rc) return rc;
    const Plan p = plan_dense(M, K, N);
    hipStream_t st = (hipStream_t)stream;
    F8Args a = {};
    a.w = (const unsigned char*)w; a.s = scales; a.e8 = e8m0; a.E = 1; a.wrows = N; a.K = K; a.N = N;
    a.x = x; a.xrows = M; a.y = y; a.rows = M; a.tm = p.tm; a.half = dtype == F16;
    if (!p.gemm) return launch_fp8_skinny(a, dtype, F8_PRODUCT, ceil_div(M, a.tm), st);
    rc = quantize_rows(a, x, dtype, M, (char*)workspace, st);
    if (rc) return rc;
    const int parts = fp8_gemm_parts(M, K, N, p.tm);
    a.partial = (float*)((char*)workspace + rows_bytes(M, K));
    a.part_ld = ceil_div(N, 4) * 4;
    return launch_fp8_gemm(a, ceil_div(M, a.tm), parts, st);
}

size_t kmi_gather_qmm_fp8_workspace_bytes(int64_t P, int64_t X, int64_t M, int64_t E, int64_t K, int64_t N,
                                          int dtype) {
    if (P <= 0 || X <= 0 || M <= 0 || E <= 0 || K <= 0 || N <= 0) return 0;
    const Plan p = plan_grouped(P * M, P, E, K, N, false);
    if (p.pairs) return 0;
    return sort_index_bytes(P * M, E, p.tm) + (p.gemm ? rows_bytes(X * M, K) : 0);
}

int kmi_gather_qmm_fp8(const void* x, int64_t X, int64_t M, int64_t K, const uint32_t* w, const void* scales,
                       int e8m0, int64_t E, int64_t N, const int32_t* lhs, const int32_t* rhs, int64_t P, int dtype,
                       void* y, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    const char* what = "gather_qmm (fp8)";
    int rc = check_operands(what, dtype, K, N, x, w);
    if (rc) return rc;
    KMI_CHECK_ARG(E > 0 && E <= MAX_E, "%s: %lld experts (1..%lld)", what, (long long)E, (long long)MAX_E);
    KMI_CHECK_ARG(X >= 1 && M >= 1 && P >= 0 && P < (1LL << 31) && M < (1LL << 31) && P * M < (1LL << 31) &&
                  X < (1LL << 31) && X * M < (1LL << 31), "%s: too many rows", what);
    if (P == 0) return OK;
    KMI_CHECK_ARG(x && w && scales && lhs && rhs && y, "%s: null pointer", what);
    const Plan p = plan_grouped(P * M, P, E, K, N, false);
    KMI_CHECK_ARG(!p.gemm || X * M * fp8_row_bytes(K) < (1LL << 31), "%s: x past 2 GiB of codes", what);
    rc = check_workspace(what, kmi_gather_qmm_fp8_workspace_bytes(P, X, M, E, K, N, dtype), workspace,
                         workspace_bytes);
    if (rc) return rc;
    hipStream_t st = (hipStream_t)stream;
    SortedRows sr = {};
    if (!p.pairs) {
        rc = launch_sort_rows(rhs, P, M, (int)E, p.tm, workspace, (uint16_t*)y, N, st, &sr);
        if (rc) return rc;
    }
    F8Args a = {};
    a.w = (const unsigned char*)w; a.s = scales; a.e8 = e8m0; a.E = E; a.wrows = N; a.K = K; a.N = N;
    a.x = x; a.xrows = X * M; a.y = y; a.rows = P * M; a.tm = p.tm; a.half = dtype == F16;
    a.tiles = sr.tiles; a.sorted = sr.sorted; a.lhs = lhs; a.lhs_div = 1; a.lhs_inv = 1.0; a.Mper = M;
    if (p.pairs) {
        a.route = rhs;
        a.tm = 1;
        return launch_fp8_skinny(a, dtype, F8_PRODUCT, P, st);
    }
    if (!p.gemm) return launch_fp8_skinny(a, dtype, F8_PRODUCT, sr.max_tiles, st);
    rc = quantize_rows(a, x, dtype, X * M, (char*)workspace + sort_index_bytes(P * M, E, p.tm), st);
    return rc ? rc : launch_fp8_gemm(a, sr.max_tiles, 1, st);
}

size_t kmi_switch_glu_fp8_workspace_bytes(int64_t T, int64_t H, int64_t I, int k, int64_t E) {
    if (T <= 0 || H <= 0 || I <= 0 || k <= 0 || E <= 0) return 0;
    const int64_t P = T * k;
    const Plan p = plan_grouped(P, P, E, H > I ? H : I, I, true);
    return align256((size_t)P * H * 2) + (p.pairs ? 0 : sort_index_bytes(P, E, p.tm)) +
           (p.gemm ? values_bytes(T, H) + rows_bytes(P, I) : align256((size_t)P * I * 2));
}

int kmi_switch_glu_fp8(const void* x, int64_t T, int64_t H, int64_t I, int k, const int32_t* inds,
                       const void* scores, const uint32_t* w_gu, const void* s_gu, const uint32_t* w_down,
                       const void* s_down, int e8m0, int64_t E, int dtype, void* out, void* workspace,
                       size_t workspace_bytes, void* stream) {
    clear_error();
    const char* what = "switch_glu (fp8)";
    KMI_CHECK_ARG(dtype == BF16, "%s: only bfloat16 activations are implemented", what);
    int rc = check_operands(what, dtype, H, 2 * I, x, w_gu);
    if (rc) return rc;
    rc = check_operands(what, dtype, I, H, workspace, w_down);
    if (rc) return rc;
    KMI_CHECK_ARG(I % F8_BLOCK == 0, "%s: I=%lld (gate and up stack in whole blocks of 128)", what, (long long)I);
    KMI_CHECK_ARG(k >= 1 && k <= 64 && E >= 1 && E <= MAX_E, "%s: top-%d of %lld experts", what, k, (long long)E);
    KMI_CHECK_ARG(T >= 0 && T < (1LL << 31) && T * k < (1LL << 31), "%s: T=%lld", what, (long long)T);
    if (T == 0) return OK;
    KMI_CHECK_ARG(x && inds && w_gu && s_gu && w_down && s_down && out, "%s: null pointer", what);
    const int64_t P = T * k;
    const Plan p = plan_grouped(P, P, E, H > I ? H : I, I, true);
    KMI_CHECK_ARG(!p.gemm || (2 * T * fp8_row_bytes(H) < (1LL << 31) && P * I < (1LL << 31)),
                  "%s: activations past 2 GiB", what);
    rc = check_workspace(what, kmi_switch_glu_fp8_workspace_bytes(T, H, I, k, E), workspace, workspace_bytes);
    if (rc) return rc;
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    uint16_t* y = scores ? (uint16_t*)ws : (uint16_t*)out;
    ws += align256((size_t)P * H * 2);
    SortedRows sr = {};
    if (!p.pairs) {
        rc = launch_sort_rows(inds, P, 1, (int)E, p.tm, ws, y, H, st, &sr);
        if (rc) return rc;
        ws += sort_index_bytes(P, E, p.tm);
    }
    F8Args g = {};
    g.w = (const unsigned char*)w_gu; g.s = s_gu; g.e8 = e8m0; g.E = E; g.wrows = 2 * I; g.K = H; g.N = I;
    g.x = x; g.xrows = T; g.rows = P; g.tm = p.tm;
    g.tiles = sr.tiles; g.sorted = sr.sorted; g.lhs_div = k; g.lhs_inv = 1.0 / k; g.Mper = 1;
    F8Args d = g;
    d.w = (const unsigned char*)w_down; d.s = s_down; d.wrows = H; d.K = I; d.N = H; d.xrows = P; d.y = y;
    d.lhs_div = 1; d.lhs_inv = 1.0;
    if (p.gemm) {
        rc = launch_fp8_rows(x, dtype, T, H, (unsigned char*)ws, nullptr, st);
        if (rc) return rc;
        g.x = ws; g.xld = 2 * fp8_row_bytes(H);
        ws += values_bytes(T, H);
        d.x = g.y = ws; d.xld = I; d.in_order = 1; d.xs_ld = g.ys_ld = fp8_row_scales(I);
        d.xs = g.ys = (unsigned char*)ws + align256((size_t)P * I);
        rc = launch_fp8_glu(g, sr.max_tiles, st);
        if (rc) return rc;
        rc = launch_fp8_gemm(d, sr.max_tiles, 1, st);
    } else {
        if (p.pairs) {
            g.route = d.route = inds;
            g.tm = d.tm = 1;
        }
        d.x = g.y = ws;
        rc = launch_fp8_skinny(g, dtype, F8_GLU, p.pairs ? P : sr.max_tiles, st);
        if (rc) return rc;
        if (p.pairs && scores && fp8_combine_supported(I, k)) return launch_fp8_combine(d, scores, k, T, out, st);
        rc = launch_fp8_skinny(d, dtype, F8_DOWN, p.pairs ? P : sr.max_tiles, st);
    }
    if (rc) return rc;
    if (scores) return kmi_moe_combine(y, scores, dtype, T, k, H, out, stream);
    return OK;
}

}  // extern "C"
