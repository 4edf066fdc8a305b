// Host side of the fp8 block-128 GEMM and of the gated feed-forward block: argument checks, tensor maps and
// launches.  Included by capi.cu, whose error, device and driver helpers it uses.
#pragma once

#include "fp8_gemm_kernels.cuh"
#include "gated_kernels.cuh"

namespace b200 {
namespace {

// Row-major matrix [rows][cols] of `elem`-byte elements with row pitch `ld` (elements) -> 2-D map, 128-byte swizzle,
// out-of-range elements read as zero and are not written.
int encode_matrix_map(CUtensorMap* map, const void* base, int elem, long long cols, long long rows, long long ld,
                      unsigned box_cols, unsigned box_rows) {
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * elem};
    cuuint32_t box[2] = {box_cols, box_rows};
    cuuint32_t step[2] = {1, 1};
    CUresult r = g_encode(map, elem == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2,
                          const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(B200_E_DRIVER, "cuTensorMapEncodeTiled (matrix) failed with CUresult %d", (int)r);
    return 0;
}

std::map<int, bool> g_dense_ready;   // devices whose kernels were given their shared memory

template <FfMode kMode> int opt_in_ff() {
    int rc = opt_in_smem(ff_gemm_pair<kMode, false>, kFfSmemBytes);
    return rc ? rc : opt_in_smem(ff_gemm_pair<kMode, true>, kFfSmemBytes);
}

// Lock, current device and per-device state of one call.
struct DenseCall {
    std::lock_guard<std::mutex> lock;
    DeviceGuard guard;
    DeviceState* st = nullptr;
    cudaStream_t stream;
    int rc;
    DenseCall(int device, void* s) : lock(g_mutex), stream(static_cast<cudaStream_t>(s)) {
        if ((rc = guard.enter(device))) return;
        // a thread that has not used CUDA yet (autograd runs backward passes on its own threads) has the device but
        // no context, which the tensor-map encoder asks for: cudaSetDevice makes the device's context current
        if ((rc = bind(device))) return;
        if ((rc = device_state(device, &st))) return;
        bool& ready = g_dense_ready[device];
        if (ready) return;
        if ((rc = opt_in_smem(fp8_gemm_pair<false>, kFp8SmemBytes))) return;
        if ((rc = opt_in_smem(fp8_gemm_pair<true>, kFp8SmemBytes))) return;
        if ((rc = opt_in_ff<FfMode::Forward>())) return;
        if ((rc = opt_in_ff<FfMode::GradHidden>())) return;
        if ((rc = opt_in_ff<FfMode::GradInput>())) return;
        if ((rc = opt_in_ff<FfMode::GradWeight>())) return;
        ready = true;
    }
    static int bind(int device) {
        B200_CUDA(cudaSetDevice(device));
        return 0;
    }
};

// Launch that may start while the kernel before it on the stream still runs (the kernel waits for it itself).
template <typename... Args>
int launch_dense(const char* name, void (*kernel)(Args...), dim3 grid, int threads, uint32_t smem, cudaStream_t stream,
                 Args... args) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    B200_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    ++g_launches;
    g_last_kernel = name;
    return 0;
}
int pair_grid(long long tiles, int sm_count) {
    const int pairs = sm_count / 2;
    return 2 * static_cast<int>(tiles < pairs ? tiles : pairs);
}

int check_dtype(const char* what, int dtype) {
    if (dtype == B200_DTYPE_F16 || dtype == B200_DTYPE_BF16) return 0;
    return fail(B200_E_VARIANT, "%s: dtype %d is neither B200_DTYPE_F16 nor B200_DTYPE_BF16", what, dtype);
}
// A matrix that TMA reads or writes: 16-byte aligned base and row pitch.
int check_matrix(const char* what, const char* name, const void* p, long long ld, long long cols, int elem) {
    if (!p) return fail(B200_E_NULL, "%s: %s is NULL", what, name);
    if (!aligned16(p)) return fail(B200_E_ALIGN, "%s: %s must be 16-byte aligned", what, name);
    if (ld < cols || (ld * elem) % 16)
        return fail(B200_E_ALIGN, "%s: row pitch %lld of %s must be at least %lld and a multiple of %d elements", what, ld, name,
                    cols, 16 / elem);
    return 0;
}
int check_positive(const char* what, int m, int n, int k) {
    if (m > 0 && n > 0 && k > 0) return 0;
    return fail(B200_E_SHAPE, "%s: m, n, k must be positive (got %d %d %d)", what, m, n, k);
}
int check_gated(const char* what, int dtype, int act, int m, int n, int k) {
    int rc = check_dtype(what, dtype);
    if (rc) return rc;
    if (act != B200_ACT_SILU && act != B200_ACT_GELU)
        return fail(B200_E_VARIANT, "%s: activation %d is neither B200_ACT_SILU nor B200_ACT_GELU", what, act);
    if ((rc = check_positive(what, m, n, k))) return rc;
    if (n % 8 || k % 8) return fail(B200_E_SHAPE, "%s: n=%d and k=%d must be multiples of 8", what, n, k);
    return 0;
}

template <FfMode kMode> int launch_ff(const char* name, FfProblem& p, int dtype, DenseCall& call, void* status) {
    p.status = status ? static_cast<uint32_t*>(status) : call.st->status;
    const int grid = pair_grid(static_cast<long long>(p.m_tiles) * p.n_tiles * p.batches, call.st->sm_count);
    if (dtype == B200_DTYPE_BF16)
        return launch_dense(name, ff_gemm_pair<kMode, true>, dim3(grid), kFfThreads, kFfSmemBytes, call.stream, p);
    return launch_dense(name, ff_gemm_pair<kMode, false>, dim3(grid), kFfThreads, kFfSmemBytes, call.stream, p);
}

// Maps and sizes that the forward pass and its recomputation share.
int ff_projections(FfProblem& p, const void* x, long long ldx, const void* w1, long long ldw1, const void* w2, long long ldw2,
                   int act, int m, int n, int k) {
    int rc;
    if ((rc = encode_matrix_map(&p.a[0], x, 2, k, m, ldx, 64, 128))) return rc;
    if ((rc = encode_matrix_map(&p.b[0], w1, 2, k, n, ldw1, 64, 128))) return rc;
    if ((rc = encode_matrix_map(&p.b[1], w2, 2, k, n, ldw2, 64, 128))) return rc;
    p.rows = m;
    p.cols = n;
    p.k_tiles = (k + 63) / 64;
    p.segments = 1;
    p.m_tiles = (m + 255) / 256;
    p.n_tiles = (n + 127) / 128;
    p.batches = 1;
    p.gelu = act == B200_ACT_GELU;
    return 0;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

int b200_fp8_quantize_rows(const void* x, int dtype, int rows, int k, int64_t ldx, void* q, int64_t ldq, float* sf,
                           int64_t sf_row, int64_t sf_col, int pow2, void* stream, int device) {
    const char* what = "fp8 quantize rows";
    int rc;
    if (!x || !sf) return fail(B200_E_NULL, "%s: NULL tensor pointer", what);
    if ((rc = check_dtype(what, dtype))) return rc;
    if ((rc = check_positive(what, rows, 1, k))) return rc;
    if (ldx < k) return fail(B200_E_ALIGN, "%s: ldx=%lld must be at least k=%d", what, (long long)ldx, k);
    if ((rc = check_matrix(what, "q", q, ldq, k, 1))) return rc;
    DenseCall call(device, stream);
    if (call.rc) return call.rc;
    const long long units = static_cast<long long>(rows) * ((k + kFp8Block - 1) / kFp8Block);
    constexpr int kPerBlock = kRowThreads / 16 * kRowUnits;
    const long long blocks = (units + kPerBlock - 1) / kPerBlock;
    if (blocks > 0x7FFFFFFFll) return fail(B200_E_LIMIT, "%s: rows=%d and k=%d are too many blocks for one launch", what, rows, k);
    const bool vec = aligned16(x) && ldx % 8 == 0;
    const uint16_t* src = static_cast<const uint16_t*>(x);
    uint8_t* qp = static_cast<uint8_t*>(q);
#define B200_ROWS(bf, p2, v)                                                                                                  \
    return launch_dense("fp8_quantize_rows", fp8_quantize_rows<bf, p2, v>, dim3(static_cast<unsigned>(blocks)), kRowThreads, \
                        0u, call.stream, src, static_cast<long long>(ldx), rows, k, qp, static_cast<long long>(ldq), sf,     \
                        static_cast<long long>(sf_row), static_cast<long long>(sf_col))
    if (dtype == B200_DTYPE_BF16) {
        if (pow2) { if (vec) B200_ROWS(true, true, true); else B200_ROWS(true, true, false); }
        else { if (vec) B200_ROWS(true, false, true); else B200_ROWS(true, false, false); }
    } else {
        if (pow2) { if (vec) B200_ROWS(false, true, true); else B200_ROWS(false, true, false); }
        else { if (vec) B200_ROWS(false, false, true); else B200_ROWS(false, false, false); }
    }
#undef B200_ROWS
}

int b200_fp8_quantize_blocks(const void* w, int dtype, int n, int k, int64_t ldw, void* q, int64_t ldq, float* sf,
                             int64_t sf_row, int64_t sf_col, void* stream, int device) {
    const char* what = "fp8 quantize blocks";
    int rc;
    if (!w || !sf) return fail(B200_E_NULL, "%s: NULL tensor pointer", what);
    if ((rc = check_dtype(what, dtype))) return rc;
    if ((rc = check_positive(what, 1, n, k))) return rc;
    if (ldw < k) return fail(B200_E_ALIGN, "%s: ldw=%lld must be at least k=%d", what, (long long)ldw, k);
    if ((rc = check_matrix(what, "q", q, ldq, k, 1))) return rc;
    if (n > 65535 * kFp8Block) return fail(B200_E_LIMIT, "%s: n=%d is more than %d", what, n, 65535 * kFp8Block);
    DenseCall call(device, stream);
    if (call.rc) return call.rc;
    const bool vec = aligned16(w) && ldw % 8 == 0;
    const dim3 grid((k + kFp8Block - 1) / kFp8Block, (n + kFp8Block - 1) / kFp8Block);
    const uint16_t* src = static_cast<const uint16_t*>(w);
    uint8_t* qp = static_cast<uint8_t*>(q);
#define B200_BLOCKS(bf, v)                                                                                               \
    return launch_dense("fp8_quantize_blocks", fp8_quantize_blocks<bf, v>, grid, 256, 0u, call.stream, src,              \
                        static_cast<long long>(ldw), n, k, qp, static_cast<long long>(ldq), sf,                          \
                        static_cast<long long>(sf_row), static_cast<long long>(sf_col))
    if (dtype == B200_DTYPE_BF16) { if (vec) B200_BLOCKS(true, true); else B200_BLOCKS(true, false); }
    else { if (vec) B200_BLOCKS(false, true); else B200_BLOCKS(false, false); }
#undef B200_BLOCKS
}

int b200_fp8_dequantize_rows(const void* q, int64_t ldq, const float* sf, int64_t sf_row, int64_t sf_col, int rows, int k,
                             int out_dtype, void* out, int64_t ldo, void* stream, int device) {
    const char* what = "fp8 dequantize rows";
    int rc;
    if (!sf || !out) return fail(B200_E_NULL, "%s: NULL tensor pointer", what);
    if ((rc = check_dtype(what, out_dtype))) return rc;
    if ((rc = check_positive(what, rows, 1, k))) return rc;
    if (ldo < k) return fail(B200_E_ALIGN, "%s: ldo=%lld must be at least k=%d", what, (long long)ldo, k);
    if ((rc = check_matrix(what, "q", q, ldq, k, 1))) return rc;
    DenseCall call(device, stream);
    if (call.rc) return call.rc;
    const long long blocks = (static_cast<long long>(rows) * ((k + 7) / 8) + 255) / 256;
    if (blocks > 0x7FFFFFFFll) return fail(B200_E_LIMIT, "%s: rows=%d and k=%d are too many for one launch", what, rows, k);
    auto* kernel = out_dtype == B200_DTYPE_BF16 ? &fp8_dequantize_rows<true> : &fp8_dequantize_rows<false>;
    return launch_dense("fp8_dequantize_rows", kernel, dim3(static_cast<unsigned>(blocks)), 256, 0u, call.stream,
                        static_cast<const uint8_t*>(q), static_cast<long long>(ldq), sf, static_cast<long long>(sf_row),
                        static_cast<long long>(sf_col), rows, k, static_cast<uint16_t*>(out), static_cast<long long>(ldo));
}

int b200_fp8_gemm(const void* a, int64_t lda, const float* sfa, int64_t sfa_row, int64_t sfa_col, const void* b, int64_t ldb,
                  const float* sfb, int64_t sfb_row, int64_t sfb_col, void* c, int64_t ldc, int out_dtype, int m, int n, int k,
                  void* stream, int device, uint32_t* status) {
    const char* what = "fp8 gemm";
    int rc;
    if (!sfa || !sfb) return fail(B200_E_NULL, "%s: NULL scale pointer", what);
    if ((rc = check_dtype(what, out_dtype))) return rc;
    if ((rc = check_positive(what, m, n, k))) return rc;
    if (n % 8) return fail(B200_E_SHAPE, "%s: n=%d is not a multiple of 8", what, n);
    if ((rc = check_matrix(what, "a", a, lda, k, 1))) return rc;
    if ((rc = check_matrix(what, "b", b, ldb, k, 1))) return rc;
    if ((rc = check_matrix(what, "c", c, ldc, n, 2))) return rc;
    DenseCall call(device, stream);
    if (call.rc) return call.rc;
    Fp8Problem p;
    if ((rc = encode_matrix_map(&p.a, a, 1, k, m, lda, 128, 128))) return rc;
    if ((rc = encode_matrix_map(&p.b, b, 1, k, n, ldb, 128, 128))) return rc;
    if ((rc = encode_matrix_map(&p.c, c, 2, n, m, ldc, 64, 32))) return rc;
    p.sfa = sfa;
    p.sfa_row = sfa_row;
    p.sfa_col = sfa_col;
    p.sfb = sfb;
    p.sfb_row = sfb_row;
    p.sfb_col = sfb_col;
    p.m = m;
    p.n = n;
    p.k_tiles = (k + kFp8Block - 1) / kFp8Block;
    p.m_tiles = (m + 255) / 256;
    p.n_tiles = (n + 255) / 256;
    p.status = status ? status : call.st->status;
    const int grid = pair_grid(static_cast<long long>(p.m_tiles) * p.n_tiles, call.st->sm_count);
    auto* kernel = out_dtype == B200_DTYPE_BF16 ? &fp8_gemm_pair<true> : &fp8_gemm_pair<false>;
    return launch_dense("fp8_gemm_pair", kernel, dim3(grid), kFp8Threads, kFp8SmemBytes, call.stream, p);
}

int b200_gated_forward(const void* x, int64_t ldx, const void* w1, int64_t ldw1, const void* w2, int64_t ldw2, int dtype, int act,
                       void* h, int64_t ldh, void* qg, void* qu, int64_t ldq, float* sg, float* su, int64_t sf_row,
                       int64_t sf_col, int m, int n, int k, void* stream, int device, uint32_t* status) {
    const char* what = "gated forward";
    int rc;
    if ((rc = check_gated(what, dtype, act, m, n, k))) return rc;
    if ((rc = check_matrix(what, "x", x, ldx, k, 2))) return rc;
    if ((rc = check_matrix(what, "w1", w1, ldw1, k, 2))) return rc;
    if ((rc = check_matrix(what, "w2", w2, ldw2, k, 2))) return rc;
    if ((rc = check_matrix(what, "h", h, ldh, n, 2))) return rc;
    const bool keep = qg != nullptr;
    if (keep) {
        if (!sg || !su) return fail(B200_E_NULL, "%s: 8-bit copies need their scales", what);
        if ((rc = check_matrix(what, "qg", qg, ldq, n, 1))) return rc;
        if ((rc = check_matrix(what, "qu", qu, ldq, n, 1))) return rc;
    }
    DenseCall call(device, stream);
    if (call.rc) return call.rc;
    FfProblem p;
    memset(&p, 0, sizeof p);
    if ((rc = ff_projections(p, x, ldx, w1, ldw1, w2, ldw2, act, m, n, k))) return rc;
    if ((rc = encode_matrix_map(&p.out[0], h, 2, n, m, ldh, 64, 32))) return rc;
    if (keep) {
        if ((rc = encode_matrix_map(&p.kept[0], qg, 1, n, m, ldq, 128, 32))) return rc;
        if ((rc = encode_matrix_map(&p.kept[1], qu, 1, n, m, ldq, 128, 32))) return rc;
        p.sf[0] = sg;
        p.sf[1] = su;
        p.sf_row = sf_row;
        p.sf_col = sf_col;
        p.keep = 1;
    }
    return launch_ff<FfMode::Forward>("ff_gemm_pair<Forward>", p, dtype, call, status);
}

int b200_gated_grad_hidden(const void* x, int64_t ldx, const void* w1, int64_t ldw1, const void* w2, int64_t ldw2, int dtype,
                           int act, const void* dh, int64_t ld_dh, void* dg, void* du, int64_t ld_out, int m, int n, int k,
                           void* stream, int device, uint32_t* status) {
    const char* what = "gated grad hidden";
    int rc;
    if ((rc = check_gated(what, dtype, act, m, n, k))) return rc;
    if ((rc = check_matrix(what, "x", x, ldx, k, 2))) return rc;
    if ((rc = check_matrix(what, "w1", w1, ldw1, k, 2))) return rc;
    if ((rc = check_matrix(what, "w2", w2, ldw2, k, 2))) return rc;
    if ((rc = check_matrix(what, "dh", dh, ld_dh, n, 2))) return rc;
    if ((rc = check_matrix(what, "dg", dg, ld_out, n, 2))) return rc;
    if ((rc = check_matrix(what, "du", du, ld_out, n, 2))) return rc;
    DenseCall call(device, stream);
    if (call.rc) return call.rc;
    FfProblem p;
    memset(&p, 0, sizeof p);
    if ((rc = ff_projections(p, x, ldx, w1, ldw1, w2, ldw2, act, m, n, k))) return rc;
    if ((rc = encode_matrix_map(&p.out[0], dg, 2, n, m, ld_out, 64, 32))) return rc;
    if ((rc = encode_matrix_map(&p.out[1], du, 2, n, m, ld_out, 64, 32))) return rc;
    p.dh = static_cast<const uint16_t*>(dh);
    p.ld_dh = ld_dh;
    return launch_ff<FfMode::GradHidden>("ff_gemm_pair<GradHidden>", p, dtype, call, status);
}

int b200_gated_grad_hidden_kept(const void* qg, const void* qu, int64_t ldq, const float* sg, const float* su, int64_t sf_row,
                                int64_t sf_col, int dtype, int act, const void* dh, int64_t ld_dh, void* dg, void* du,
                                int64_t ld_out, int m, int n, void* stream, int device) {
    const char* what = "gated grad hidden (kept)";
    int rc;
    if ((rc = check_gated(what, dtype, act, m, n, 8))) return rc;
    if (!sg || !su) return fail(B200_E_NULL, "%s: NULL scale pointer", what);
    if ((rc = check_matrix(what, "qg", qg, ldq, n, 1))) return rc;
    if ((rc = check_matrix(what, "qu", qu, ldq, n, 1))) return rc;
    if ((rc = check_matrix(what, "dh", dh, ld_dh, n, 2))) return rc;
    if ((rc = check_matrix(what, "dg", dg, ld_out, n, 2))) return rc;
    if ((rc = check_matrix(what, "du", du, ld_out, n, 2))) return rc;
    DenseCall call(device, stream);
    if (call.rc) return call.rc;
    const long long blocks = (static_cast<long long>(m) * (n / 8) + 256 * kKeptUnits - 1) / (256 * kKeptUnits);
    if (blocks > 0x7FFFFFFFll) return fail(B200_E_LIMIT, "%s: m=%d and n=%d are too many for one launch", what, m, n);
    auto* kernel = dtype == B200_DTYPE_BF16 ? &gated_grad_kept<true> : &gated_grad_kept<false>;
    return launch_dense("gated_grad_kept", kernel, dim3(static_cast<unsigned>(blocks)), 256, 0u, call.stream,
                        static_cast<const uint8_t*>(qg), static_cast<const uint8_t*>(qu), static_cast<long long>(ldq), sg, su,
                        static_cast<long long>(sf_row), static_cast<long long>(sf_col), static_cast<const uint16_t*>(dh),
                        static_cast<long long>(ld_dh), static_cast<uint16_t*>(dg), static_cast<uint16_t*>(du),
                        static_cast<long long>(ld_out), m, n, act == B200_ACT_GELU ? 1 : 0);
}

int b200_gated_grad_input(const void* dg, const void* du, int64_t ld_g, const void* w1, int64_t ldw1, const void* w2,
                          int64_t ldw2, int dtype, void* dx, int64_t ld_dx, int m, int n, int k, void* stream, int device,
                          uint32_t* status) {
    const char* what = "gated grad input";
    int rc;
    if ((rc = check_gated(what, dtype, B200_ACT_SILU, m, n, k))) return rc;
    if ((rc = check_matrix(what, "dg", dg, ld_g, n, 2))) return rc;
    if ((rc = check_matrix(what, "du", du, ld_g, n, 2))) return rc;
    if ((rc = check_matrix(what, "w1", w1, ldw1, k, 2))) return rc;
    if ((rc = check_matrix(what, "w2", w2, ldw2, k, 2))) return rc;
    if ((rc = check_matrix(what, "dx", dx, ld_dx, k, 2))) return rc;
    DenseCall call(device, stream);
    if (call.rc) return call.rc;
    FfProblem p;
    memset(&p, 0, sizeof p);
    if ((rc = encode_matrix_map(&p.a[0], dg, 2, n, m, ld_g, 64, 128))) return rc;
    if ((rc = encode_matrix_map(&p.a[1], du, 2, n, m, ld_g, 64, 128))) return rc;
    if ((rc = encode_matrix_map(&p.b[0], w1, 2, k, n, ldw1, 64, 64))) return rc;
    if ((rc = encode_matrix_map(&p.b[1], w2, 2, k, n, ldw2, 64, 64))) return rc;
    if ((rc = encode_matrix_map(&p.out[0], dx, 2, k, m, ld_dx, 64, 32))) return rc;
    p.rows = m;
    p.cols = k;
    p.k_tiles = (n + 63) / 64;
    p.segments = 2;
    p.m_tiles = (m + 255) / 256;
    p.n_tiles = (k + 255) / 256;
    p.batches = 1;
    return launch_ff<FfMode::GradInput>("ff_gemm_pair<GradInput>", p, dtype, call, status);
}

int b200_gated_grad_weight(const void* dg, const void* du, int64_t ld_g, const void* x, int64_t ldx, int dtype, void* dw1,
                           void* dw2, int64_t ld_dw, int m, int n, int k, void* stream, int device, uint32_t* status) {
    const char* what = "gated grad weight";
    int rc;
    if ((rc = check_gated(what, dtype, B200_ACT_SILU, m, n, k))) return rc;
    if ((rc = check_matrix(what, "dg", dg, ld_g, n, 2))) return rc;
    if ((rc = check_matrix(what, "du", du, ld_g, n, 2))) return rc;
    if ((rc = check_matrix(what, "x", x, ldx, k, 2))) return rc;
    if ((rc = check_matrix(what, "dw1", dw1, ld_dw, k, 2))) return rc;
    if ((rc = check_matrix(what, "dw2", dw2, ld_dw, k, 2))) return rc;
    DenseCall call(device, stream);
    if (call.rc) return call.rc;
    FfProblem p;
    memset(&p, 0, sizeof p);
    if ((rc = encode_matrix_map(&p.a[0], dg, 2, n, m, ld_g, 64, 64))) return rc;
    if ((rc = encode_matrix_map(&p.a[1], du, 2, n, m, ld_g, 64, 64))) return rc;
    if ((rc = encode_matrix_map(&p.b[0], x, 2, k, m, ldx, 64, 64))) return rc;
    if ((rc = encode_matrix_map(&p.out[0], dw1, 2, k, n, ld_dw, 64, 32))) return rc;
    if ((rc = encode_matrix_map(&p.out[1], dw2, 2, k, n, ld_dw, 64, 32))) return rc;
    p.rows = n;
    p.cols = k;
    p.k_tiles = (m + 63) / 64;
    p.segments = 1;
    p.m_tiles = (n + 255) / 256;
    p.n_tiles = (k + 255) / 256;
    p.batches = 2;
    return launch_ff<FfMode::GradWeight>("ff_gemm_pair<GradWeight>", p, dtype, call, status);
}

}  // extern "C"
