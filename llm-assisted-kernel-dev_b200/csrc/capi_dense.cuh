// Host side of the fp8 block-128 GEMM and of the gated feed-forward block: argument checks, tensor maps and
// launches.  Included by capi.cu, whose error, device and driver helpers it uses.
#pragma once

#include "fp8_gemm_kernels.cuh"
#include "few_tokens_kernels.cuh"

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
    int rc;
    if ((rc = opt_in_smem(ff_gemm_pair<kMode, false, 256>, ff_smem_bytes<256>()))) return rc;
    if ((rc = opt_in_smem(ff_gemm_pair<kMode, true, 256>, ff_smem_bytes<256>()))) return rc;
    if ((rc = opt_in_smem(ff_gemm_pair<kMode, false, 128>, ff_smem_bytes<128>()))) return rc;
    return opt_in_smem(ff_gemm_pair<kMode, true, 128>, ff_smem_bytes<128>());
}

template <FewOp kOp, int kTokens, bool kFuse = false> int opt_in_few() {
    int rc = opt_in_smem(few_tokens_gemm<kOp, kTokens, false, kFuse>, few_smem_bytes<kOp, kTokens, kFuse>());
    return rc ? rc : opt_in_smem(few_tokens_gemm<kOp, kTokens, true, kFuse>, few_smem_bytes<kOp, kTokens, kFuse>());
}
template <FewOp kOp> int opt_in_few_all() {
    int rc;
    if ((rc = opt_in_few<kOp, 16>())) return rc;
    if ((rc = opt_in_few<kOp, 32>())) return rc;
    if ((rc = opt_in_few<kOp, 64>())) return rc;
    return opt_in_few<kOp, 128>();
}

template <typename K> int load_kernel(K kernel) {
    cudaFuncAttributes attr;
    B200_CUDA(cudaFuncGetAttributes(&attr, kernel));
    return 0;
}
// Kernels without a shared-memory opt-in are loaded here rather than by their first launch, which may be captured.
int load_streaming() {
    int rc;
    if ((rc = load_kernel(fp8_quantize_rows<true, true, true>)) || (rc = load_kernel(fp8_quantize_rows<true, true, false>)) ||
        (rc = load_kernel(fp8_quantize_rows<true, false, true>)) || (rc = load_kernel(fp8_quantize_rows<true, false, false>)) ||
        (rc = load_kernel(fp8_quantize_rows<false, true, true>)) || (rc = load_kernel(fp8_quantize_rows<false, true, false>)) ||
        (rc = load_kernel(fp8_quantize_rows<false, false, true>)) || (rc = load_kernel(fp8_quantize_rows<false, false, false>)) ||
        (rc = load_kernel(fp8_quantize_blocks<true, true>)) || (rc = load_kernel(fp8_quantize_blocks<true, false>)) ||
        (rc = load_kernel(fp8_quantize_blocks<false, true>)) || (rc = load_kernel(fp8_quantize_blocks<false, false>)) ||
        (rc = load_kernel(fp8_dequantize_rows<true>)) || (rc = load_kernel(fp8_dequantize_rows<false>)) ||
        (rc = load_kernel(gated_grad_kept<true>)) || (rc = load_kernel(gated_grad_kept<false>))) return rc;
    return 0;
}

// Lock, current device and per-device state of one call.
struct DenseCall {
    std::lock_guard<std::mutex> lock;
    DeviceGuard guard;
    DeviceState* st = nullptr;
    cudaStream_t stream;
    int device;
    int rc;
    DenseCall(int device_, void* s) : lock(g_mutex), stream(static_cast<cudaStream_t>(s)), device(device_) {
        if ((rc = guard.enter(device))) return;
        // a thread that has not used CUDA yet (autograd runs backward passes on its own threads) has the device but
        // no context, which the tensor-map encoder asks for: cudaSetDevice makes the device's context current
        if ((rc = bind(device))) return;
        bool& ready = g_dense_ready[device];
        if (!ready && (rc = reject_first_capture())) return;
        if ((rc = device_state(device, &st)) || ready) return;
        if ((rc = opt_in_smem(fp8_gemm_pair<false, 256>, fp8_smem_bytes<256>()))) return;
        if ((rc = opt_in_smem(fp8_gemm_pair<true, 256>, fp8_smem_bytes<256>()))) return;
        if ((rc = opt_in_smem(fp8_gemm_pair<false, 128>, fp8_smem_bytes<128>()))) return;
        if ((rc = opt_in_smem(fp8_gemm_pair<true, 128>, fp8_smem_bytes<128>()))) return;
        if ((rc = opt_in_few_all<FewOp::Few8>())) return;
        if ((rc = opt_in_few_all<FewOp::FewGated>())) return;
        if ((rc = opt_in_few<FewOp::Few8, 16, true>())) return;
        if ((rc = opt_in_ff<FfMode::Forward>())) return;
        if ((rc = opt_in_smem(ff_forward_keep<false>, ff_smem_bytes<256>()))) return;
        if ((rc = opt_in_smem(ff_forward_keep<true>, ff_smem_bytes<256>()))) return;
        if ((rc = opt_in_ff<FfMode::GradHidden>())) return;
        if ((rc = opt_in_ff<FfMode::GradInput>())) return;
        if ((rc = opt_in_ff<FfMode::GradWeight>())) return;
        if ((rc = load_streaming())) return;
        ready = true;
    }
    // The one-time set-up of a device loads code and clears state, which a capture does not allow.
    int reject_first_capture() {
        cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
        B200_CUDA(cudaStreamIsCapturing(stream, &cs));
        if (cs == cudaStreamCaptureStatusNone) return 0;
        return fail(B200_E_CAPTURE, "the stream is being captured and this is the first call on its device: make one call outside "
                                    "the capture first");
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

template <FfMode kMode> int launch_ff(const char* name, FfProblem& p, int tile_n, int dtype, DenseCall& call, void* status) {
    p.status = status ? static_cast<uint32_t*>(status) : call.st->status;
    const int grid = pair_grid(static_cast<long long>(p.m_tiles) * p.n_tiles * p.batches, call.st->sm_count);
    const bool bf16 = dtype == B200_DTYPE_BF16;
    if (tile_n == 128)
        return launch_dense(name, bf16 ? &ff_gemm_pair<kMode, true, 128> : &ff_gemm_pair<kMode, false, 128>, dim3(grid), kFfThreads,
                            ff_smem_bytes<128>(), call.stream, p);
    return launch_dense(name, bf16 ? &ff_gemm_pair<kMode, true, 256> : &ff_gemm_pair<kMode, false, 256>, dim3(grid), kFfThreads,
                        ff_smem_bytes<256>(), call.stream, p);
}

// A 128-wide tile's time in hundredths of a 256-wide one's (measured: gated 62 to 68, fp8 62 to 68; m=512 n=4096 k=7168 fp8, one
// round either way: 20.8 us with 128-wide tiles, 26.9 with 256-wide ones).
constexpr long long kFfNarrowCost = 65, kFp8NarrowCost = 68;
// Width of the merged B: 128 where whole rounds of 256-wide tiles over the CTA pairs cost more.  `row_tiles` counts every batch.
int pair_tile_n(int row_tiles, int cols256, int cols128, long long narrow_cost, int sm_count) {
    const int pairs = sm_count / 2;
    const long long wide = (static_cast<long long>(row_tiles) * cols256 + pairs - 1) / pairs;
    const long long narrow = (static_cast<long long>(row_tiles) * cols128 + pairs - 1) / pairs;
    return narrow * narrow_cost < wide * 100 ? 128 : 256;
}

// CTAs that share the k range of one tile: as many as give every tile's cluster a place at the same time, with at least four
// steps each.  `places[i]`: clusters of 1 << i CTAs that have one.
int few_splits(long long tiles, int steps, const int (&places)[4]) {
    int i = 3;
    while (i > 0 && (tiles > places[i] || steps < (4 << i))) --i;
    return 1 << i;
}

template <FewOp kOp, int kTokens, bool kBf16, bool kFuse = false> int launch_few_as(FewProblem& p, DenseCall& call) {
    using S = FewShape<kOp, kTokens, kFuse>;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cfg.blockDim = dim3(S::kThreads, 1, 1);
    cfg.dynamicSmemBytes = few_smem_bytes<kOp, kTokens, kFuse>();
    cfg.stream = call.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    struct Places { int of[4] = {0, 0, 0, 0}; };
    static std::map<int, Places> known;      // by device; guarded by the call's lock
    Places& places = known[call.device];
    if (!places.of[0]) {
        cfg.numAttrs = 1;
        // One CTA per SM: what the GPU holds, which for clusters of eight is less than its SMs make up (a GPC's SMs are no multiple
        // of eight): 16 tiles (n=2048 k=4096, 128 tokens) took 15.2 us in two rounds of eights, 8.7 in one of fours.  Two CTAs per
        // SM: their number; a cluster or two that start late cost less than halving the loads in flight (32 tiles, n=4096
        // k=7168: one token 10.6 us with eights, 13.7 with fours).
        for (int i = 3; i >= 0; --i) {       // the first entry last: it marks the row as complete
            if (S::kCtasPerSm == 2) {
                places.of[i] = call.st->sm_count * 2 >> i;
                continue;
            }
            attr[0].val.clusterDim.x = 1 << i;
            cfg.gridDim = dim3(1 << i, 1, 1);
            B200_CUDA(cudaOccupancyMaxActiveClusters(&places.of[i], few_tokens_gemm<kOp, kTokens, kBf16, kFuse>, &cfg));
        }
    }
    const int tiles = (p.n + 127) / 128, token_tiles = (p.m + kTokens - 1) / kTokens;
    const int splits = few_splits(static_cast<long long>(tiles) * token_tiles, p.steps, places.of);
    cfg.gridDim = dim3(tiles * splits, token_tiles, 1);
    attr[0].val.clusterDim.x = splits;
    cfg.numAttrs = 2;
    B200_CUDA(cudaLaunchKernelEx(&cfg, few_tokens_gemm<kOp, kTokens, kBf16, kFuse>, p));
    ++g_launches;
    g_last_kernel = kOp == FewOp::Few8 ? "few_tokens_gemm<Few8>" : "few_tokens_gemm<FewGated>";
    return 0;
}
// The token tile: the smallest that holds all tokens, up to 128.
int few_tokens_tile(int m) { return m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128; }
template <FewOp kOp> int launch_few(FewProblem& p, int dtype, DenseCall& call, uint32_t* status) {
    p.status = status ? status : call.st->status;
    const bool bf16 = dtype == B200_DTYPE_BF16;
    switch (few_tokens_tile(p.m)) {
        case 16: return bf16 ? launch_few_as<kOp, 16, true>(p, call) : launch_few_as<kOp, 16, false>(p, call);
        case 32: return bf16 ? launch_few_as<kOp, 32, true>(p, call) : launch_few_as<kOp, 32, false>(p, call);
        case 64: return bf16 ? launch_few_as<kOp, 64, true>(p, call) : launch_few_as<kOp, 64, false>(p, call);
        default: return bf16 ? launch_few_as<kOp, 128, true>(p, call) : launch_few_as<kOp, 128, false>(p, call);
    }
}
// Whether the few-token kernel or the CTA-pair kernel is faster.  Up to 64 rows always the former.  Beyond, its tiles are
// 128 x 128; it gains while several CTAs can share the k range of each and k is long enough to pay for the exchange.  Measured,
// few-token against pair, us:
//   fp8    n=4096 k=7168: m=128 (32 tiles) 12.9 / 20.1, m=256 (64) 16.4 / 20.2, m=512 (128) 33.6 / 20.9; n=4096 k=2048: m=128
//          8.0 / 8.4, m=256 8.7 / 8.5; n=2048 k=1024: m=128 6.2 / 5.7, m=512 7.0 / 6.0
//   gated  n=4096 k=7168: m=128 (32) 26.7 / 31.5, m=256 (64) 33.2 / 32.2; n=2048 k=4096: m=256 (32) 14.2 / 16.8, m=512 (64) 19.6 /
//          18.3; n=2048 k=1024: m=128 8.6 / 7.3
bool few_is_faster(FewOp op, int m, int n, int k, int sm_count) {
    if (m <= 64) return true;
    const long long tiles = static_cast<long long>((n + 127) / 128) * ((m + 127) / 128);
    return k >= 2048 && (op == FewOp::Few8 ? 2 : 4) * tiles <= sm_count;
}
constexpr int kFuseMost = 16;            // rows up to which fp8_linear quantises inside the product's kernel

// Maps and sizes that the forward pass and its recomputation share.
int ff_projections(FfProblem& p, int* tile_n, const void* x, long long ldx, const void* w1, long long ldw1, const void* w2,
                   long long ldw2, int act, int m, int n, int k, bool keep, int sm_count) {
    int rc;
    p.m_tiles = (m + 255) / 256;
    // 8-bit copies are made from whole 128-wide blocks
    *tile_n = keep ? 256 : pair_tile_n(p.m_tiles, (n + 127) / 128, (n + 63) / 64, kFfNarrowCost, sm_count);
    const int cols = *tile_n / 2;
    if ((rc = encode_matrix_map(&p.a[0], x, 2, k, m, ldx, 64, 128))) return rc;
    if ((rc = encode_matrix_map(&p.b[0], w1, 2, k, n, ldw1, 64, cols))) return rc;
    if ((rc = encode_matrix_map(&p.b[1], w2, 2, k, n, ldw2, 64, cols))) return rc;
    p.rows = m;
    p.cols = n;
    p.k_tiles = (k + 63) / 64;
    p.segments = 1;
    p.n_tiles = (n + cols - 1) / cols;
    p.batches = 1;
    p.gelu = act == B200_ACT_GELU;
    return 0;
}

int quantize_rows_launch(const char* what, const void* x, int dtype, int rows, int k, long long ldx, void* q, long long ldq,
                         float* sf, long long sf_row, long long sf_col, int pow2, DenseCall& call) {
    const long long units = static_cast<long long>(rows) * ((k + kFp8Block - 1) / kFp8Block);
    constexpr int kPerBlock = kRowThreads / kRowLanes * kRowUnits;
    const long long blocks = (units + kPerBlock - 1) / kPerBlock;
    if (units + kPerBlock > 0xFFFFFFFFll) return fail(B200_E_LIMIT, "%s: %d rows and k=%d are too many blocks", what, rows, k);
    const bool vec = aligned16(x) && ldx % 8 == 0;
    const uint16_t* src = static_cast<const uint16_t*>(x);
    uint8_t* qp = static_cast<uint8_t*>(q);
    auto go = [&](auto* kernel) {
        return launch_dense("fp8_quantize_rows", kernel, dim3(static_cast<unsigned>(blocks)), kRowThreads, 0u, call.stream, src, ldx,
                            rows, k, qp, ldq, sf, sf_row, sf_col);
    };
    if (dtype == B200_DTYPE_BF16) {
        if (pow2) return vec ? go(&fp8_quantize_rows<true, true, true>) : go(&fp8_quantize_rows<true, true, false>);
        return vec ? go(&fp8_quantize_rows<true, false, true>) : go(&fp8_quantize_rows<true, false, false>);
    }
    if (pow2) return vec ? go(&fp8_quantize_rows<false, true, true>) : go(&fp8_quantize_rows<false, true, false>);
    return vec ? go(&fp8_quantize_rows<false, false, true>) : go(&fp8_quantize_rows<false, false, false>);
}

int dequantize_rows_launch(const char* what, const void* q, long long ldq, const float* sf, long long sf_row, long long sf_col,
                           int rows, int k, int out_dtype, void* out, long long ldo, DenseCall& call) {
    const long long blocks = (static_cast<long long>(rows) * ((k + 15) / 16) + 255) / 256;
    if (blocks * 256 > 0xFFFFFFFFll) return fail(B200_E_LIMIT, "%s: %d rows and k=%d are too many", what, rows, k);
    auto* kernel = out_dtype == B200_DTYPE_BF16 ? &fp8_dequantize_rows<true> : &fp8_dequantize_rows<false>;
    return launch_dense("fp8_dequantize_rows", kernel, dim3(static_cast<unsigned>(blocks)), 256, 0u, call.stream,
                        static_cast<const uint8_t*>(q), ldq, sf, sf_row, sf_col, rows, k, static_cast<uint16_t*>(out), ldo);
}

// What the gated block keeps in 8 bits, one buffer: codes of g, u [m, n] and, on request, x [m, k] (row pitches padded to
// 16 bytes), then their power-of-two scales, block by block.
struct Kept {
    uint8_t *qg, *qu, *qx;
    float *sg, *su, *sx;
    long long ldn, ldk;
    size_t bytes;
    Kept(void* base, int m, int n, int k, bool with_x) {
        ldn = (n + 15) / 16 * 16;
        ldk = (k + 15) / 16 * 16;
        const size_t codes = static_cast<size_t>(m) * ldn, codes_x = with_x ? static_cast<size_t>(m) * ldk : 0;
        const size_t scales = static_cast<size_t>(m) * ((n + kFp8Block - 1) / kFp8Block);
        const size_t scales_x = with_x ? static_cast<size_t>(m) * ((k + kFp8Block - 1) / kFp8Block) : 0;
        qg = static_cast<uint8_t*>(base);
        qu = qg + codes;
        qx = qu + codes;
        sg = reinterpret_cast<float*>(qx + codes_x);
        su = sg + scales;
        sx = su + scales;
        bytes = 2 * codes + codes_x + 4 * (2 * scales + scales_x);
    }
};

// One quantised operand: codes, row pitch, scales and their strides.
struct Fp8Matrix {
    const void* q;
    long long ld;
    const float* sf;
    long long sf_row, sf_col;
};
// Codes of [m, k] in the linear layer's scratch, the scales behind them.
size_t fp8_codes_bytes(int m, int k) { return static_cast<size_t>(m) * ((k + 15) / 16 * 16); }

// `after_quantiser`: the launch before this one on the stream is fp8_quantize_rows, which has waited for all before it
// by the time this kernel starts and does not write the weights.
int fp8_gemm_launch(const Fp8Matrix& a, const Fp8Matrix& b, void* c, long long ldc, int out_dtype, int m, int n, int k,
                    bool after_quantiser, DenseCall& call, uint32_t* status) {
    int rc;
    if (few_is_faster(FewOp::Few8, m, n, k, call.st->sm_count)) {
        FewProblem p;
        memset(&p, 0, sizeof p);
        if ((rc = encode_matrix_map(&p.w[0], b.q, 1, k, n, b.ld, 128, 128))) return rc;
        if ((rc = encode_matrix_map(&p.x, a.q, 1, k, m, a.ld, 128, few_tokens_tile(m)))) return rc;
        p.sfa = a.sf;
        p.sfa_row = a.sf_row;
        p.sfa_col = a.sf_col;
        p.sfb = b.sf;
        p.sfb_row = b.sf_row;
        p.sfb_col = b.sf_col;
        p.c = static_cast<uint16_t*>(c);
        p.ldc = ldc;
        p.m = m;
        p.n = n;
        p.steps = (k + kFp8Block - 1) / kFp8Block;
        p.weights_early = after_quantiser;
        return launch_few<FewOp::Few8>(p, out_dtype, call, status);
    }
    Fp8Problem p;
    if ((rc = encode_matrix_map(&p.a, a.q, 1, k, m, a.ld, 128, 128))) return rc;
    p.m_tiles = (m + 255) / 256;
    const int tile_n = pair_tile_n(p.m_tiles, (n + 255) / 256, (n + 127) / 128, kFp8NarrowCost, call.st->sm_count);
    if ((rc = encode_matrix_map(&p.b, b.q, 1, k, n, b.ld, 128, tile_n / 2))) return rc;
    if ((rc = encode_matrix_map(&p.c, c, 2, n, m, ldc, 64, 32))) return rc;
    p.sfa = a.sf;
    p.sfa_row = a.sf_row;
    p.sfa_col = a.sf_col;
    p.sfb = b.sf;
    p.sfb_row = b.sf_row;
    p.sfb_col = b.sf_col;
    p.m = m;
    p.n = n;
    p.k_tiles = (k + kFp8Block - 1) / kFp8Block;
    p.n_tiles = (n + tile_n - 1) / tile_n;
    p.status = status ? status : call.st->status;
    const int grid = pair_grid(static_cast<long long>(p.m_tiles) * p.n_tiles, call.st->sm_count);
    const bool bf16 = out_dtype == B200_DTYPE_BF16;
    if (tile_n == 128)
        return launch_dense("fp8_gemm_pair", bf16 ? &fp8_gemm_pair<true, 128> : &fp8_gemm_pair<false, 128>, dim3(grid), kFp8Threads,
                            fp8_smem_bytes<128>(), call.stream, p);
    return launch_dense("fp8_gemm_pair", bf16 ? &fp8_gemm_pair<true, 256> : &fp8_gemm_pair<false, 256>, dim3(grid), kFp8Threads,
                        fp8_smem_bytes<256>(), call.stream, p);
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
    return quantize_rows_launch(what, x, dtype, rows, k, ldx, q, ldq, sf, sf_row, sf_col, pow2, call);
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
    return dequantize_rows_launch(what, q, ldq, sf, sf_row, sf_col, rows, k, out_dtype, out, ldo, call);
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
    const Fp8Matrix ma{a, lda, sfa, sfa_row, sfa_col}, mb{b, ldb, sfb, sfb_row, sfb_col};
    return fp8_gemm_launch(ma, mb, c, ldc, out_dtype, m, n, k, false, call, status);
}

size_t b200_fp8_linear_scratch_bytes(int m, int k) {
    if (m <= kFuseMost || k <= 0) return 0;          // quantised on the way into the product
    return fp8_codes_bytes(m, k) + static_cast<size_t>(m) * ((k + kFp8Block - 1) / kFp8Block) * 4;
}

int b200_fp8_linear(const void* x, int64_t ldx, int dtype, const void* w, int64_t ldw, const float* sfw, int64_t sfw_row,
                    int64_t sfw_col, void* y, int64_t ldy, int m, int n, int k, void* scratch, size_t scratch_bytes,
                    void* stream, int device, uint32_t* status) {
    const char* what = "fp8 linear";
    int rc;
    if (!x || !sfw) return fail(B200_E_NULL, "%s: NULL tensor pointer", what);
    if ((rc = check_dtype(what, dtype))) return rc;
    if ((rc = check_positive(what, m, n, k))) return rc;
    if (n % 8) return fail(B200_E_SHAPE, "%s: n=%d is not a multiple of 8", what, n);
    if (ldx < k) return fail(B200_E_ALIGN, "%s: ldx=%lld must be at least k=%d", what, (long long)ldx, k);
    if ((rc = check_matrix(what, "w", w, ldw, k, 1))) return rc;
    if ((rc = check_matrix(what, "y", y, ldy, n, 2))) return rc;
    if (m > kFuseMost && (!scratch || !aligned16(scratch) || scratch_bytes < b200_fp8_linear_scratch_bytes(m, k)))
        return fail(B200_E_WORKSPACE, "%s: needs %zu scratch bytes, 16-byte aligned", what, b200_fp8_linear_scratch_bytes(m, k));
    DenseCall call(device, stream);
    if (call.rc) return call.rc;
    if (m <= kFuseMost) {
        FewProblem p;
        memset(&p, 0, sizeof p);
        if ((rc = encode_matrix_map(&p.w[0], w, 1, k, n, ldw, 128, 128))) return rc;
        p.x16 = static_cast<const uint16_t*>(x);
        p.ldx = ldx;
        p.k = k;
        p.vec = aligned16(x) && ldx % 8 == 0;
        p.sfb = sfw;
        p.sfb_row = sfw_row;
        p.sfb_col = sfw_col;
        p.c = static_cast<uint16_t*>(y);
        p.ldc = ldy;
        p.m = m;
        p.n = n;
        p.steps = (k + kFp8Block - 1) / kFp8Block;
        p.status = status ? status : call.st->status;
        return dtype == B200_DTYPE_BF16 ? launch_few_as<FewOp::Few8, 16, true, true>(p, call)
                                        : launch_few_as<FewOp::Few8, 16, false, true>(p, call);
    }
    uint8_t* q = static_cast<uint8_t*>(scratch);
    float* sf = reinterpret_cast<float*>(q + fp8_codes_bytes(m, k));
    const int64_t ldq = (k + 15) / 16 * 16;
    if ((rc = quantize_rows_launch(what, x, dtype, m, k, ldx, q, ldq, sf, 1, m, 0, call))) return rc;
    const Fp8Matrix ma{q, ldq, sf, 1, m}, mb{w, ldw, sfw, sfw_row, sfw_col};
    return fp8_gemm_launch(ma, mb, y, ldy, dtype, m, n, k, true, call, status);
}

size_t b200_gated_kept_bytes(int m, int n, int k, int keep_x) {
    if (m <= 0 || n <= 0 || k <= 0) return 0;
    return Kept(nullptr, m, n, k, keep_x != 0).bytes;
}

size_t b200_gated_backward_scratch_bytes(int m, int n, int k, int kept) {
    if (m <= 0 || n <= 0 || k <= 0) return 0;
    return static_cast<size_t>(m) * n * 4 + (kept ? static_cast<size_t>(m) * k * 2 : 0);
}

int b200_gated_forward(const void* x, int64_t ldx, const void* w1, int64_t ldw1, const void* w2, int64_t ldw2, int dtype, int act,
                       void* h, int64_t ldh, void* kept, size_t kept_bytes, int keep_x, int m, int n, int k, void* stream,
                       int device, uint32_t* status) {
    const char* what = "gated forward";
    int rc;
    if ((rc = check_gated(what, dtype, act, m, n, k))) return rc;
    if ((rc = check_matrix(what, "x", x, ldx, k, 2))) return rc;
    if ((rc = check_matrix(what, "w1", w1, ldw1, k, 2))) return rc;
    if ((rc = check_matrix(what, "w2", w2, ldw2, k, 2))) return rc;
    if ((rc = check_matrix(what, "h", h, ldh, n, 2))) return rc;
    if (kept && (!aligned16(kept) || kept_bytes < b200_gated_kept_bytes(m, n, k, keep_x)))
        return fail(B200_E_WORKSPACE, "%s: the 8-bit copies need %zu bytes, 16-byte aligned", what, b200_gated_kept_bytes(m, n, k, keep_x));
    DenseCall call(device, stream);
    if (call.rc) return call.rc;
    if (!kept && few_is_faster(FewOp::FewGated, m, n, k, call.st->sm_count)) {
        FewProblem f;
        memset(&f, 0, sizeof f);
        if ((rc = encode_matrix_map(&f.w[0], w1, 2, k, n, ldw1, 64, 128))) return rc;
        if ((rc = encode_matrix_map(&f.w[1], w2, 2, k, n, ldw2, 64, 128))) return rc;
        if ((rc = encode_matrix_map(&f.x, x, 2, k, m, ldx, 64, few_tokens_tile(m)))) return rc;
        f.c = static_cast<uint16_t*>(h);
        f.ldc = ldh;
        f.m = m;
        f.n = n;
        f.steps = (k + 63) / 64;
        f.gelu = act == B200_ACT_GELU;
        return launch_few<FewOp::FewGated>(f, dtype, call, status);
    }
    FfProblem p;
    memset(&p, 0, sizeof p);
    int tile_n;
    if ((rc = ff_projections(p, &tile_n, x, ldx, w1, ldw1, w2, ldw2, act, m, n, k, kept != nullptr, call.st->sm_count))) return rc;
    if ((rc = encode_matrix_map(&p.out[0], h, 2, n, m, ldh, 64, 32))) return rc;
    if (kept) {
        const Kept v(kept, m, n, k, keep_x != 0);
        if ((rc = encode_matrix_map(&p.kept[0], v.qg, 1, n, m, v.ldn, 128, 32))) return rc;
        if ((rc = encode_matrix_map(&p.kept[1], v.qu, 1, n, m, v.ldn, 128, 32))) return rc;
        p.sf[0] = v.sg;
        p.sf[1] = v.su;
        p.sf_row = 1;
        p.sf_col = m;
        if (keep_x && (rc = quantize_rows_launch(what, x, dtype, m, k, ldx, v.qx, v.ldk, v.sx, 1, m, 1, call))) return rc;
        p.status = status ? status : call.st->status;
        auto* kernel = dtype == B200_DTYPE_BF16 ? &ff_forward_keep<true> : &ff_forward_keep<false>;
        return launch_dense("ff_forward_keep", kernel, dim3(pair_grid(static_cast<long long>(p.m_tiles) * p.n_tiles, call.st->sm_count)),
                            kKeepThreads, ff_smem_bytes<256>(), call.stream, p);
    }
    return launch_ff<FfMode::Forward>("ff_gemm_pair<Forward>", p, tile_n, dtype, call, status);
}

int b200_gated_backward(const void* x, int64_t ldx, const void* kept, size_t kept_bytes, int keep_x, const void* w1, int64_t ldw1,
                        const void* w2, int64_t ldw2, int dtype, int act, const void* dh, int64_t ld_dh, void* dx, int64_t ld_dx,
                        void* dw1, void* dw2, int64_t ld_dw, int m, int n, int k, void* scratch, size_t scratch_bytes,
                        void* stream, int device, uint32_t* status) {
    const char* what = "gated backward";
    int rc;
    const bool weights = dw1 || dw2;
    if ((rc = check_gated(what, dtype, act, m, n, k))) return rc;
    if (!dx && !weights) return fail(B200_E_NULL, "%s: no gradient is asked for", what);
    if (!kept && (rc = check_matrix(what, "x", x, ldx, k, 2))) return rc;
    if ((rc = check_matrix(what, "w1", w1, ldw1, k, 2))) return rc;
    if ((rc = check_matrix(what, "w2", w2, ldw2, k, 2))) return rc;
    if ((rc = check_matrix(what, "dh", dh, ld_dh, n, 2))) return rc;
    if (dx && (rc = check_matrix(what, "dx", dx, ld_dx, k, 2))) return rc;
    if (dw1 && (rc = check_matrix(what, "dw1", dw1, ld_dw, k, 2))) return rc;
    if (dw2 && (rc = check_matrix(what, "dw2", dw2, ld_dw, k, 2))) return rc;
    if (kept && (!aligned16(kept) || kept_bytes < b200_gated_kept_bytes(m, n, k, keep_x)))
        return fail(B200_E_WORKSPACE, "%s: the 8-bit copies are %zu bytes, 16-byte aligned", what, b200_gated_kept_bytes(m, n, k, keep_x));
    if (kept && weights && !keep_x) return fail(B200_E_VARIANT, "%s: the weights' gradients need an 8-bit copy of x (keep_x)", what);
    const size_t need = b200_gated_backward_scratch_bytes(m, n, k, kept != nullptr);
    if (!scratch || !aligned16(scratch) || scratch_bytes < need)
        return fail(B200_E_WORKSPACE, "%s: needs %zu scratch bytes, 16-byte aligned", what, need);
    DenseCall call(device, stream);
    if (call.rc) return call.rc;
    uint16_t* dg = static_cast<uint16_t*>(scratch);
    uint16_t* du = dg + static_cast<size_t>(m) * n;
    // the gradients of the two projections
    if (kept) {
        const Kept v(const_cast<void*>(kept), m, n, k, keep_x != 0);
        const unsigned row_groups = static_cast<unsigned>((m + kKeptRows - 1) / kKeptRows);
        const unsigned column_blocks = (n + kKeptCols - 1) / kKeptCols;
        const unsigned most = std::max(1u, call.st->sm_count * kKeptBlocksPerSm / column_blocks);
        const dim3 grid(column_blocks, std::min(std::min(row_groups, most), 65535u));
        auto* kernel = dtype == B200_DTYPE_BF16 ? &gated_grad_kept<true> : &gated_grad_kept<false>;
        if ((rc = launch_dense("gated_grad_kept", kernel, grid, kKeptThreads, 0u, call.stream, (const uint8_t*)v.qg, (const uint8_t*)v.qu,
                               v.ldn, (const float*)v.sg, (const float*)v.su, 1ll, (long long)m, static_cast<const uint16_t*>(dh),
                               static_cast<long long>(ld_dh), dg, du, (long long)n, m, n, act == B200_ACT_GELU ? 1 : 0))) return rc;
        if (weights) {      // x back to 16 bits, exactly: an operand of the weights' gradients
            uint16_t* x16 = du + static_cast<size_t>(m) * n;
            if ((rc = dequantize_rows_launch(what, v.qx, v.ldk, v.sx, 1, m, m, k, dtype, x16, k, call))) return rc;
            x = x16;
            ldx = k;
        }
    } else {
        FfProblem p;
        memset(&p, 0, sizeof p);
        int tile_n;
        if ((rc = ff_projections(p, &tile_n, x, ldx, w1, ldw1, w2, ldw2, act, m, n, k, false, call.st->sm_count))) return rc;
        if ((rc = encode_matrix_map(&p.out[0], dg, 2, n, m, n, 64, 32))) return rc;
        if ((rc = encode_matrix_map(&p.out[1], du, 2, n, m, n, 64, 32))) return rc;
        p.dh = static_cast<const uint16_t*>(dh);
        p.ld_dh = ld_dh;
        if ((rc = launch_ff<FfMode::GradHidden>("ff_gemm_pair<GradHidden>", p, tile_n, dtype, call, status))) return rc;
    }
    if (dx) {
        FfProblem p;
        memset(&p, 0, sizeof p);
        if ((rc = encode_matrix_map(&p.a[0], dg, 2, n, m, n, 64, 128))) return rc;
        if ((rc = encode_matrix_map(&p.a[1], du, 2, n, m, n, 64, 128))) return rc;
        if ((rc = encode_matrix_map(&p.b[0], w1, 2, k, n, ldw1, 64, 64))) return rc;
        if ((rc = encode_matrix_map(&p.b[1], w2, 2, k, n, ldw2, 64, 64))) return rc;
        if ((rc = encode_matrix_map(&p.out[0], dx, 2, k, m, ld_dx, 64, 32))) return rc;
        p.rows = m;
        p.cols = k;
        p.k_tiles = (n + 63) / 64;
        p.segments = 2;
        p.m_tiles = (m + 255) / 256;
        p.batches = 1;
        const int tile_n = pair_tile_n(p.m_tiles, (k + 255) / 256, (k + 127) / 128, kFfNarrowCost, call.st->sm_count);
        p.n_tiles = (k + tile_n - 1) / tile_n;
        if ((rc = launch_ff<FfMode::GradInput>("ff_gemm_pair<GradInput>", p, tile_n, dtype, call, status))) return rc;
    }
    if (weights) {
        FfProblem p;
        memset(&p, 0, sizeof p);
        p.batches = 0;
        for (int i = 0; i < 2; ++i) {      // one launch for what is asked for
            void* out = i == 0 ? dw1 : dw2;
            if (!out) continue;
            if ((rc = encode_matrix_map(&p.a[p.batches], i == 0 ? dg : du, 2, n, m, n, 64, 64))) return rc;
            if ((rc = encode_matrix_map(&p.out[p.batches], out, 2, k, n, ld_dw, 64, 32))) return rc;
            ++p.batches;
        }
        if ((rc = encode_matrix_map(&p.b[0], x, 2, k, m, ldx, 64, 64))) return rc;
        p.rows = n;
        p.cols = k;
        p.k_tiles = (m + 63) / 64;
        p.segments = 1;
        p.m_tiles = (n + 255) / 256;
        const int tile_n = pair_tile_n(p.m_tiles * p.batches, (k + 255) / 256, (k + 127) / 128, kFfNarrowCost, call.st->sm_count);
        p.n_tiles = (k + tile_n - 1) / tile_n;
        if ((rc = launch_ff<FfMode::GradWeight>("ff_gemm_pair<GradWeight>", p, tile_n, dtype, call, status))) return rc;
    }
    return 0;
}

}  // extern "C"
