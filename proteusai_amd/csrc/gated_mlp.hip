// The gated feed-forward block, forward and backward, a call per direction (gfx950).
//
//   z = x W^T + b = (gate | value),   h = act(gate) * value,   y = h Wo^T + bo
//   dh = dy Wo,   dz = (dh * value * act'(gate) | dh * act(gate)),   dx = dz W,   dW = dz^T x,   dWo = dy^T h,   db, dbo = column sums of dz and dy
//
// bf16: the products of gated_mlp_bf16.hip, with the element-wise parts and the column sums of dz as their epilogues.  fp32: the products of gemm_f32.hip with the
// element-wise parts as theirs, and the column sums and the shares of the gradients of weights added up in one launch behind them: a training pass of 2048 rows, d_model 512,
// hidden 2048 286 us where it was 304 with launches of their own for all these (286 to 319 from card to card), for 38.7 GFLOP: 121 to 135 TFLOP/s (gemm_f32.hip's large products 185).
// A forward without a backward takes 98 us at 2048 rows and 306 at 8192 (132 and 168 TFLOP/s); it writes z, too, which nothing reads then.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "gated_mlp_internal.h"
#include "gemm_f32_internal.h"

namespace {

using namespace proteus_gated;

constexpr int THREADS = 256;

// h from z, fp32, where the product cannot do it
__global__ __launch_bounds__(THREADS)
void gate_kernel(const float* __restrict__ z, float* __restrict__ h, const int64_t n, const int F, const int act)
{
    for (int64_t i = ((int64_t)blockIdx.x * THREADS + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * THREADS * 4) {
        const int64_t row = i / F;
        const float* const at = z + row * F + i;    // (2 row F + column)
        const float4 g = *reinterpret_cast<const float4*>(at), v = *reinterpret_cast<const float4*>(at + F);
        float o[4], s;
        activate<true>(act, g.x, o[0], s); activate<true>(act, g.y, o[1], s); activate<true>(act, g.z, o[2], s); activate<true>(act, g.w, o[3], s);
        *reinterpret_cast<float4*>(h + i) = make_float4(o[0] * v.x, o[1] * v.y, o[2] * v.z, o[3] * v.w);
    }
}

struct Sizes {
    int64_t rows;
    int D, F, O, type;
    size_t item() const { return type == PROTEUS_DTYPE_F32 ? 4 : 2; }
    bool taken() const
    {
        const int per = type == PROTEUS_DTYPE_F32 ? 4 : 8;
        if ((type != PROTEUS_DTYPE_F32 && type != PROTEUS_DTYPE_BF16) || rows <= 0 || D <= 0 || F <= 0 || O <= 0 || D % per || F % per || O % per) return false;
        const int most = D > O ? (D > 2 * (int64_t)F ? D : 2 * F) : (O > 2 * (int64_t)F ? O : 2 * F);
        if (F > (1 << 20) || D > (1 << 20) || O > (1 << 20) || rows > (1 << 28)) return false;
        if (type == PROTEUS_DTYPE_F32) return (rows + 512) * most * 4 < (1LL << 31) && (2LL * F + 512) * D * 4 < (1LL << 31) && ((int64_t)O + 512) * F * 4 < (1LL << 31);
        // (the paired weight's offsets in 31 bits, tiles numbered in as many)
        return 4LL * F * D < (1LL << 31) && ((rows + 127) / 128) * ((most + 127) / 128) < (1 << 28) && ((most + 127LL) / 128) * ((most + 127) / 128) * 16 < (1 << 28);
    }
};

size_t up(const size_t n) { return (n + 255) & ~(size_t)255; }

// Where things lie in the backward's workspace.
struct Layout {
    size_t dz, part, columns, total;
    size_t part_out, part_in, part_columns;         // of the gradients of Wo and of W, whose shares are added up together, and of column sums (bf16: dy's)
    Behind b;                                       // bf16
    Layout(const Sizes& s) : part_out(0), part_in(0), part_columns(0), b()
    {
        const int M = (int)s.rows;
        dz = 0;
        part = up(s.rows * 2 * s.F * s.item());
        if (s.type == PROTEUS_DTYPE_F32) {
            part_out = up(proteus_gemm_f32_workspace_bytes(s.O, s.F, M, PROTEUS_GEMM_TN));
            part_in = up(proteus_gemm_f32_workspace_bytes(2 * s.F, s.D, M, PROTEUS_GEMM_TN));
            const size_t a = proteus_train_workspace_bytes(M, 2 * s.F), c = proteus_train_workspace_bytes(M, s.O);
            part_columns = up(a > c ? a : c);
            columns = total = part + part_out + part_in + part_columns;
            return;
        }
        b = behind(M, s.D, s.F, s.O);
        part_out = up(b.part[0]);
        part_in = up(b.part[1]);
        columns = part + part_out + part_in + up(b.part[2]);
        part_columns = up((size_t)column_shares(s.rows) * s.O * 4);
        total = columns + part_columns + up((size_t)column_rows(M, s.F, s.O) * 2 * s.F * 4);
    }
};

bool off(const void* p, const uintptr_t by) { return ((uintptr_t)p & (by - 1)) != 0; }

unsigned blocks_of(const int64_t n) { const int64_t b = (n / 4 + THREADS - 1) / THREADS; return (unsigned)(b < 8192 ? b : 8192); }

#define TRY(call) do { const int rc_ = (call); if (rc_) return rc_; } while (0)

int check(const Sizes& s, const void* x, const void* const* params, const void* y, const void* kept, const size_t kept_bytes, const void* ws, const size_t ws_bytes, const size_t need, const int act)
{
    if (s.type != PROTEUS_DTYPE_F32 && s.type != PROTEUS_DTYPE_BF16) return PROTEUS_ERR_BAD_OPERAND_TYPE;
    if (act < PROTEUS_ACT_SILU || act > PROTEUS_ACT_SIGMOID) return PROTEUS_ERR_UNSUPPORTED;
    if (!x || !params || !params[0] || !params[2] || !y || (need && !ws)) return PROTEUS_ERR_NULL_POINTER;
    if (!s.taken()) return PROTEUS_ERR_BAD_SHAPE;
    for (int i = 0; i < 4; ++i) if (off(params[i], 16)) return PROTEUS_ERR_BAD_ALIGNMENT;
    if (off(x, 16) || off(y, 16) || off(kept, 256) || off(ws, 256)) return PROTEUS_ERR_BAD_ALIGNMENT;
    if ((kept && kept_bytes < proteus_gated_mlp_kept_bytes((long)s.rows, s.D, s.F, s.O, s.type)) || ws_bytes < need) return PROTEUS_ERR_TOO_LARGE;
    return 0;
}

}  // namespace

extern "C" size_t proteus_gated_mlp_kept_bytes(long rows, int d_in, int hidden, int d_out, int dtype)
{
    const Sizes s = {rows, d_in, hidden, d_out, dtype};
    return s.taken() ? up(s.rows * 2 * s.F * s.item()) + up(s.rows * s.F * s.item()) + (dtype == PROTEUS_DTYPE_BF16 ? up(s.rows * s.F) : 0) : 0;
}
extern "C" size_t proteus_gated_mlp_fwd_bytes(long rows, int d_in, int hidden, int d_out, int dtype)
{
    const Sizes s = {rows, d_in, hidden, d_out, dtype};
    if (!s.taken()) return 0;
    return up(s.rows * s.F * s.item()) + (dtype == PROTEUS_DTYPE_F32 ? up(s.rows * 2 * s.F * 4) : up(product_bytes(PROTEUS_GEMM_NT, (int)rows, d_out, hidden)));
}
extern "C" size_t proteus_gated_mlp_train_fwd_bytes(long rows, int d_in, int hidden, int d_out, int dtype)
{
    const Sizes s = {rows, d_in, hidden, d_out, dtype};
    return s.taken() && dtype == PROTEUS_DTYPE_BF16 ? up(product_bytes(PROTEUS_GEMM_NT, (int)rows, d_out, hidden)) : 0;
}
extern "C" size_t proteus_gated_mlp_bwd_bytes(long rows, int d_in, int hidden, int d_out, int dtype)
{
    const Sizes s = {rows, d_in, hidden, d_out, dtype};
    return s.taken() ? Layout(s).total : 0;
}

extern "C" int proteus_gated_mlp_fwd(const void* x, const void* const* params, void* y, void* kept, size_t kept_bytes, void* ws, size_t ws_bytes,
                                     long rows, int d_in, int hidden, int d_out, int act, int dtype, void* stream)
{
    const Sizes s = {rows, d_in, hidden, d_out, dtype};
    TRY(check(s, x, params, y, kept, kept_bytes, ws, ws_bytes, kept ? proteus_gated_mlp_train_fwd_bytes(rows, d_in, hidden, d_out, dtype) : proteus_gated_mlp_fwd_bytes(rows, d_in, hidden, d_out, dtype), act));
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int M = (int)rows, D = d_in, F = hidden, O = d_out;
    if (dtype == PROTEUS_DTYPE_F32) {
        float* const z = static_cast<float*>(kept ? kept : ws);
        float* const h = z + up(s.rows * 2 * F * 4) / 4;
        const float *X = static_cast<const float*>(x), *W = static_cast<const float*>(params[0]), *b = static_cast<const float*>(params[1]);
        if (proteus_gemm::gemm_gated_fused(M, F, D)) TRY(proteus_gemm::gemm_gated(X, W, b, nullptr, h, z, M, F, D, proteus_gemm::GATED, act, stream));
        else {
            TRY(proteus_gemm_f32(X, W, b, nullptr, z, nullptr, M, 2 * F, D, D, D, 2 * F, PROTEUS_GEMM_NT, PROTEUS_GEMM_F32, stream));
            hipLaunchKernelGGL(gate_kernel, dim3(blocks_of(s.rows * F)), dim3(THREADS), 0, st, z, h, s.rows * F, F, act);
            TRY((int)hipGetLastError());
        }
        return proteus_gemm_f32(h, static_cast<const float*>(params[2]), static_cast<const float*>(params[3]), nullptr, y, nullptr, M, O, F, F, F, O, PROTEUS_GEMM_NT, PROTEUS_GEMM_F32, stream);
    }
    uint16_t* const z = static_cast<uint16_t*>(kept);
    uint16_t* const h = kept ? z + up(s.rows * 2 * F * 2) / 2 : static_cast<uint16_t*>(ws);
    Product p = {};
    p.A = static_cast<const uint16_t*>(x); p.B = static_cast<const uint16_t*>(params[0]); p.bias = static_cast<const uint16_t*>(params[1]);
    p.C = h; p.z = z; p.rest = kept ? reinterpret_cast<uint8_t*>(h + up(s.rows * F * 2) / 2) : nullptr;
    p.M = M; p.N = F; p.K = D; p.lda = D; p.ldb = D; p.ldc = F;
    p.form = PROTEUS_GEMM_NT; p.epilogue = kept ? GATED_KEPT : GATED; p.act = act;
    Ends ends = {};
    TRY(product(p, ends, st));
    p.A = h; p.B = static_cast<const uint16_t*>(params[2]); p.bias = static_cast<const uint16_t*>(params[3]);
    p.C = static_cast<uint16_t*>(y); p.z = nullptr;
    p.N = O; p.K = F; p.lda = F; p.ldb = F; p.ldc = O;
    p.epilogue = PLAIN; p.part = reinterpret_cast<float*>(static_cast<char*>(ws) + (kept ? 0 : up(s.rows * F * 2)));
    TRY(product(p, ends, st));
    return finish(ends, st);
}

extern "C" int proteus_gated_mlp_bwd(const void* x, const void* const* params, const void* dy, void* dx, void* const* grads, const void* kept, size_t kept_bytes, void* ws, size_t ws_bytes,
                                     long rows, int d_in, int hidden, int d_out, int act, int dtype, void* stream)
{
    const Sizes s = {rows, d_in, hidden, d_out, dtype};
    if (!grads || !kept) return PROTEUS_ERR_NULL_POINTER;
    TRY(check(s, x, params, dy, kept, kept_bytes, ws, ws_bytes, 1, act));
    const Layout at(s);
    if (ws_bytes < at.total) return PROTEUS_ERR_TOO_LARGE;
    if (off(dx, 16)) return PROTEUS_ERR_BAD_ALIGNMENT;
    for (int i = 0; i < 4; ++i) if (off(grads[i], 16)) return PROTEUS_ERR_BAD_ALIGNMENT;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int M = (int)rows, D = d_in, F = hidden, O = d_out;
    char* const w = static_cast<char*>(ws);
    const bool inner = dx || grads[0] || grads[1];
    if (dtype == PROTEUS_DTYPE_F32) {
        const float *z = static_cast<const float*>(kept), *h = z + up(s.rows * 2 * F * 4) / 4, *d = static_cast<const float*>(dy), *W = static_cast<const float*>(params[0]),
                    *Wo = static_cast<const float*>(params[2]);
        float* const dz = reinterpret_cast<float*>(w + at.dz);
        // what is left to add up, column sums and shares of the gradients of weights, in one launch at the end where it can be
        proteus_gemm::PendingSums sums;
        char* const part = w + at.part;
        if (grads[2]) TRY(proteus_gemm::gemm_begin(d, h, static_cast<float*>(grads[2]), O, F, M, O, F, F, part, at.part_out, sums, stream));
        if (grads[3] && !sums.add({d, static_cast<float*>(grads[3]), M, O})) TRY(proteus_colsum(d, static_cast<float*>(grads[3]), part + at.part_out + at.part_in, at.part_columns, (long)rows, O, stream));
        if (inner) {
            TRY(proteus_gemm::gemm_gated(d, Wo, nullptr, z, dz, nullptr, M, F, O, proteus_gemm::GATED_GRAD, act, stream));
            if (grads[1] && !sums.add({dz, static_cast<float*>(grads[1]), M, 2 * F}))
                TRY(proteus_colsum(dz, static_cast<float*>(grads[1]), part + at.part_out + at.part_in, at.part_columns, (long)rows, 2 * F, stream));
            if (grads[0]) TRY(proteus_gemm::gemm_begin(dz, static_cast<const float*>(x), static_cast<float*>(grads[0]), 2 * F, D, M, 2 * F, D, D, part + at.part_out, at.part_in, sums, stream));
            if (dx) TRY(proteus_gemm_f32(dz, W, nullptr, nullptr, dx, nullptr, M, D, 2 * F, 2 * F, D, D, PROTEUS_GEMM_NN, PROTEUS_GEMM_F32, stream));
        }
        return proteus_gemm::gemm_sums(sums, stream);
    }
    uint16_t *z = const_cast<uint16_t*>(static_cast<const uint16_t*>(kept)), *h = z + up(s.rows * 2 * F * 2) / 2, *dz = reinterpret_cast<uint16_t*>(w + at.dz);
    float* const columns = reinterpret_cast<float*>(w + at.columns + at.part_columns);
    const uint16_t* const d = static_cast<const uint16_t*>(dy);
    Ends ends = {};
    auto of = [&](const int form, const uint16_t* A, const uint16_t* B, void* C, const int m, const int n, const int k, const int64_t lda, const size_t part) {
        Product p = {};
        p.A = A; p.B = B; p.C = static_cast<uint16_t*>(C);
        p.M = m; p.N = n; p.K = k; p.lda = lda; p.ldb = n; p.ldc = n;
        p.form = form; p.epilogue = PLAIN; p.part = reinterpret_cast<float*>(w + part);
        return p;
    };
    if (inner) {
        Product p = of(PROTEUS_GEMM_NN, d, static_cast<const uint16_t*>(params[2]), dz, M, F, O, O, at.part);
        p.epilogue = GATED_GRAD; p.act = act;
        p.z = z; p.rest = reinterpret_cast<uint8_t*>(h + up(s.rows * F * 2) / 2);
        p.columns = grads[1] ? columns : nullptr;
        TRY(product(p, ends, st));
        if (grads[1]) ends.columns[ends.column_count++] = {columns, static_cast<uint16_t*>(grads[1]), column_rows(M, F, O), 2 * F};
    }
    const Product last[3] = {of(PROTEUS_GEMM_TN, d, h, grads[2], O, F, M, O, at.part), of(PROTEUS_GEMM_TN, dz, static_cast<const uint16_t*>(x), grads[0], 2 * F, D, M, 2 * F, at.part + at.part_out),
                             of(PROTEUS_GEMM_NN, dz, static_cast<const uint16_t*>(params[0]), dx, M, D, 2 * F, 2 * F, at.part + at.part_out + at.part_in)};
    const Columns columns_of_dy = {grads[3] ? d : nullptr, reinterpret_cast<float*>(w + at.columns), static_cast<uint16_t*>(grads[3]), rows, O};
    TRY(products_behind(at.b, last, columns_of_dy, ends, st));
    return finish(ends, st);
}
