// Linear layers on gfx950: a matrix product with bias, activation and residual in its epilogue, dense or with one weight
// matrix per modality over rows sorted by modality, and its gradients.
//
//   z = x W^T + b,  y = act(z) + residual             act: none, relu, gelu (erf), silu
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz
//
// Types float, bfloat16, half; sums are float.  z is kept for the backward pass in the layers' type when there is an
// activation: one rounding, half a step of the type relative to z, and act' is taken at that point.
#include "linear_kernel.h"

// [rows, cols] with leading dimension ld -> the same with leading dimension ldo: operands whose rows do not start on a 4-byte
// boundary (the LDS loads' unit) are laid out anew first
template <typename T>
__global__ __launch_bounds__(256) void k_linear_relayout(const T *__restrict__ in, int64_t rows, int cols, int64_t ld,
                                                         T *__restrict__ out, int64_t ldo) {
    const int64_t n = rows * cols;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / cols, c = i - r * cols;
        out[r * ldo + c] = in[r * ld + c];
    }
}

// dz = g * act'(z), eight columns a thread.  HBM-bound: g and z are read, dz is written.
template <typename T>
__global__ __launch_bounds__(256) void k_linear_act_grad(const T *__restrict__ g, const T *__restrict__ z, int64_t rows, int cols,
                                                         int act, const int32_t *offsets, int n_sets, T *__restrict__ dz,
                                                         int64_t ldo, int vec) {
    if (offsets != nullptr) {
        const int64_t end = offsets[n_sets];
        rows = end < rows ? (end < 0 ? 0 : end) : rows;
    }
    if (vec) {
        typedef T t8 __attribute__((ext_vector_type(8)));
        const int64_t n = rows * (cols / 8);
        const int per = cols / 8;
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
            const t8 gv = reinterpret_cast<const t8 *>(g)[i], zv = reinterpret_cast<const t8 *>(z)[i];
            t8 o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = from_f32<T>(to_f32(gv[e]) * lin_slope(to_f32(zv[e]), act));
            const int64_t r = i / per, c = i - r * per;
            *reinterpret_cast<t8 *>(dz + r * ldo + c * 8) = o;
        }
    } else {
        const int64_t n = rows * cols;
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
            const int64_t r = i / cols, c = i - r * cols;
            dz[r * ldo + c] = from_f32<T>(to_f32(g[i]) * lin_slope(to_f32(z[i]), act));
        }
    }
}

// the parts of a split weight gradient, added in their order
template <typename T>
__global__ __launch_bounds__(256) void k_linear_join(const float *__restrict__ partial, int splits, int64_t n, T *__restrict__ out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float s = 0.f;
        for (int p = 0; p < splits; ++p) s += partial[(int64_t)p * n + i];
        out[i] = from_f32<T>(s);
    }
}

// rows behind the last set have no gradient: out = g there is none, g elsewhere
template <typename T>
__global__ __launch_bounds__(256) void k_linear_mask_rows(const T *__restrict__ g, int64_t rows, int cols, const int32_t *offsets,
                                                          int n_sets, T *__restrict__ out) {
    int64_t end = offsets[n_sets];
    end = end < 0 ? 0 : (end < rows ? end : rows);
    const int64_t n = rows * cols, held = end * cols;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
        out[i] = i < held ? g[i] : (T)0.f;
}

namespace {

int elem_size(int dtype) { return dtype == MTP_FLOAT ? 4 : 2; }
int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
unsigned grid_for(int64_t items) {
    const int64_t b = (items + 255) / 256;
    return (unsigned)(b < 1 ? 1 : (b > 256 * 16 ? 256 * 16 : b));
}

// rows of a 16-bit operand have to start on 4 bytes; a row distance beyond 2^20 elements would leave the loads' 32-bit offsets
bool needs_relayout(int dtype, const void *p, int64_t ld) {
    return ld > (1 << 20) || (elem_size(dtype) == 2 && (ld % 2 != 0 || (uintptr_t)p % 4 != 0));
}
int64_t relayout_bytes(int dtype, const void *p, int64_t ld, int64_t rows, int64_t cols) {
    return needs_relayout(dtype, p, ld) ? round_up(rows * round_up(cols, 8) * elem_size(dtype), 256) : 0;
}

template <typename T>
int relayout(const void **p, int64_t *ld, int64_t rows, int cols, char **ws, hipStream_t s) {
    const int dtype = sizeof(T) == 4 ? MTP_FLOAT : MTP_BFLOAT16;
    const int64_t bytes = relayout_bytes(dtype, *p, *ld, rows, cols);
    if (bytes == 0) return MTP_OK;
    const int64_t ldo = round_up(cols, 8);
    T *to = reinterpret_cast<T *>(*ws);
    hipLaunchKernelGGL(k_linear_relayout<T>, dim3(grid_for(rows * cols)), dim3(256), 0, s, reinterpret_cast<const T *>(*p), rows,
                       cols, *ld, to, ldo);
    MTP_LAUNCH_CHECK();
    *p = to;
    *ld = ldo;
    *ws += bytes;
    return MTP_OK;
}

int splits_for(int64_t rows, int in, int out, int n_sets, int dtype) {
    const int64_t tiles = (int64_t)n_sets * ((out + 127) / 128) * ((in + 127) / 128);
    const int64_t mean = rows / n_sets;
    int64_t s = (512 + tiles - 1) / tiles;
    const int64_t most = mean / (4 * 128 / elem_size(dtype));
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s);
}

template <typename T, int MODE, int BC, int BR, int WC, int WR>
int launch_tile(LinArgs a, hipStream_t s) {
    constexpr int NT = 64 * (BC / WC) * (BR / WR);
    constexpr int LDS = 2 * (BC + BR) * 128;
    a.col_tiles = (a.cols + BC - 1) / BC;
    int64_t blocks;
    if (MODE == LIN_GRAD_WEIGHT) {
        a.row_tiles = (a.out_rows + BR - 1) / BR;
        blocks = a.row_tiles * a.col_tiles * a.splits * a.n_sets;
    } else {
        // a set's last tile may be ragged, and so may the one behind the last set
        a.row_tiles = a.offsets == nullptr ? (a.rows + BR - 1) / BR : (a.rows + (int64_t)(a.n_sets + 1) * (BR - 1)) / BR;
        blocks = a.row_tiles * a.col_tiles;
    }
    MTP_REQUIRE(blocks <= 0x7fffffff, "mtp_linear: %lld workgroups are too many", (long long)blocks);
    if (blocks == 0) return MTP_OK;
    MTP_SET_MAX_LDS_ONCE((k_linear_tile<T, MODE, BC, BR, WC, WR>), LDS);
    hipLaunchKernelGGL((k_linear_tile<T, MODE, BC, BR, WC, WR>), dim3((unsigned)blocks), dim3(NT), LDS, s, a);
    MTP_LAUNCH_CHECK();
    return MTP_OK;
}

template <typename T, int MODE>
int launch_product(const LinArgs &a, hipStream_t s) {
    const int64_t r = MODE == LIN_GRAD_WEIGHT ? (int64_t)a.out_rows * a.n_sets * a.splits : a.rows;
    const int64_t big = ((r + 127) / 128) * ((a.cols + 127) / 128);
    if (big >= 256 && (a.offsets == nullptr || MODE == LIN_GRAD_WEIGHT || a.rows / a.n_sets >= 128))
        return launch_tile<T, MODE, 128, 128, 64, 64>(a, s);
    return launch_tile<T, MODE, 64, 64, 32, 32>(a, s);
}

int check_sizes(const char *who, int dtype, int64_t rows, int in, int out, const int32_t *offsets, int n_sets) {
    MTP_REQUIRE(dtype == MTP_FLOAT || dtype == MTP_BFLOAT16 || dtype == MTP_HALF, "%s: unknown type %d", who, dtype);
    MTP_REQUIRE(rows >= 0 && rows <= 0x7fffffff && in >= 1 && out >= 1 && in <= 65536 && out <= 65536,
                "%s: bad shape rows=%lld in=%d out=%d", who, (long long)rows, in, out);
    MTP_REQUIRE(n_sets >= 1 && n_sets <= 65536 && (offsets != nullptr || n_sets == 1), "%s: bad number of sets %d", who, n_sets);
    return MTP_OK;
}

template <typename T>
int forward(const void *x, int64_t rows, int in, int64_t ldx, const void *w, int out, const void *bias, int act,
            const void *residual, int64_t ldr, const int32_t *offsets, int n_sets, void *y, void *pre, char *ws, hipStream_t s) {
    int64_t ldw = in;
    int rc = relayout<T>(&x, &ldx, rows, in, &ws, s);
    if (rc == MTP_OK) rc = relayout<T>(&w, &ldw, (int64_t)n_sets * out, in, &ws, s);
    if (rc != MTP_OK) return rc;
    LinArgs a{};
    a.P = LinOperand{w, ldw, (int64_t)out * ldw};
    a.Q = LinOperand{x, ldx, 0};
    a.rows = rows;
    a.cols = out;
    a.k = in;
    a.offsets = offsets;
    a.n_sets = n_sets;
    a.bias = bias;
    a.residual = residual;
    a.ld_res = ldr;
    a.act = act;
    a.out = y;
    a.pre = pre;
    return launch_product<T, LIN_FORWARD>(a, s);
}

// where the parts of a backward pass lie in the workspace: dz, then what the products need one after the other
struct BackwardPlan {
    int64_t lddz, dz_bytes, input_bytes, weight_bytes;
    int64_t total() const { return dz_bytes + (input_bytes > weight_bytes ? input_bytes : weight_bytes); }
};
BackwardPlan plan_backward(int dtype, int64_t rows, int in, int out, int n_sets, int act, const void *g, const void *w, const void *x,
                           int64_t ldx, bool want_x, bool want_w) {
    BackwardPlan p{};
    // dz has rows of its own, so they can start where the loads want them
    const bool own = act != LIN_NONE;
    p.lddz = own && elem_size(dtype) == 2 && out % 2 != 0 ? round_up(out, 8) : out;
    p.dz_bytes = own ? round_up(rows * p.lddz * elem_size(dtype), 256) : 0;
    const void *dz = own ? nullptr : g;
    if (want_x) p.input_bytes = mtp_linear_workspace_bytes(dtype, MTP_LINEAR_GRAD_INPUT, rows, in, out, n_sets, dz, p.lddz, w, in);
    if (want_w) p.weight_bytes = mtp_linear_workspace_bytes(dtype, MTP_LINEAR_GRAD_WEIGHT, rows, in, out, n_sets, dz, p.lddz, x, ldx);
    return p;
}

template <typename T>
int grad_input(const void *dz, int64_t rows, int out, int64_t lddz, const void *w, int in, const int32_t *offsets, int n_sets,
               void *dx, char *ws, hipStream_t s) {
    int64_t ldw = in;
    int rc = relayout<T>(&dz, &lddz, rows, out, &ws, s);
    if (rc == MTP_OK) rc = relayout<T>(&w, &ldw, (int64_t)n_sets * out, in, &ws, s);
    if (rc != MTP_OK) return rc;
    LinArgs a{};
    a.P = LinOperand{w, ldw, (int64_t)out * ldw};
    a.Q = LinOperand{dz, lddz, 0};
    a.rows = rows;
    a.cols = in;
    a.k = out;
    a.offsets = offsets;
    a.n_sets = n_sets;
    a.out = dx;
    return launch_product<T, LIN_GRAD_INPUT>(a, s);
}

template <typename T>
int grad_weight(const void *dz, int64_t rows, int out, int64_t lddz, const void *x, int in, int64_t ldx, const int32_t *offsets,
                int n_sets, void *dw, void *db, char *ws, hipStream_t s) {
    int rc = relayout<T>(&dz, &lddz, rows, out, &ws, s);
    if (rc == MTP_OK) rc = relayout<T>(&x, &ldx, rows, in, &ws, s);
    if (rc != MTP_OK) return rc;
    LinArgs a{};
    a.P = LinOperand{x, ldx, 0};
    a.Q = LinOperand{dz, lddz, 0};
    a.rows = rows;
    a.cols = in;
    a.out_rows = out;
    a.offsets = offsets;
    a.n_sets = n_sets;
    a.k = (int)rows;
    a.splits = splits_for(rows, in, out, n_sets, sizeof(T) == 4 ? MTP_FLOAT : MTP_BFLOAT16);
    a.out = dw;
    a.bias_out = db;
    a.partial = reinterpret_cast<float *>(ws);
    rc = launch_product<T, LIN_GRAD_WEIGHT>(a, s);
    if (rc != MTP_OK || a.splits == 1) return rc;
    const int64_t n = (int64_t)n_sets * out * in;
    hipLaunchKernelGGL(k_linear_join<T>, dim3(grid_for(n)), dim3(256), 0, s, a.partial, a.splits, n, reinterpret_cast<T *>(dw));
    MTP_LAUNCH_CHECK();
    if (db != nullptr) {
        const int64_t m = (int64_t)n_sets * out;
        hipLaunchKernelGGL(k_linear_join<T>, dim3(grid_for(m)), dim3(256), 0, s, a.partial + (int64_t)a.splits * n, a.splits, m,
                           reinterpret_cast<T *>(db));
        MTP_LAUNCH_CHECK();
    }
    return MTP_OK;
}

}  // namespace

#define MTP_BY_TYPE(dtype, call)                              \
    ((dtype) == MTP_FLOAT ? call<float> : (dtype) == MTP_BFLOAT16 ? call<__bf16> : call<_Float16>)

extern "C" int64_t mtp_linear_workspace_bytes(int dtype, int step, int64_t rows, int in, int out, int n_sets, const void *a,
                                              int64_t lda, const void *b, int64_t ldb) {
    if (rows < 0 || in < 1 || out < 1 || n_sets < 1) return 0;
    const int64_t w_rows = (int64_t)n_sets * out;
    if (step == MTP_LINEAR_FORWARD) return relayout_bytes(dtype, a, lda, rows, in) + relayout_bytes(dtype, b, in, w_rows, in);
    if (step == MTP_LINEAR_GRAD_INPUT) return relayout_bytes(dtype, a, lda, rows, out) + relayout_bytes(dtype, b, in, w_rows, in);
    int64_t n = relayout_bytes(dtype, a, lda, rows, out) + relayout_bytes(dtype, b, ldb, rows, in);
    const int s = splits_for(rows, in, out, n_sets, dtype);
    if (s > 1) n += (int64_t)s * w_rows * (in + 1) * 4;
    return n;
}

extern "C" int mtp_linear(int dtype, const void *x, int64_t rows, int in, int64_t ldx, const void *w, int out, const void *bias,
                          int act, const void *residual, int64_t ldr, const int32_t *offsets, int n_sets, void *y, void *pre,
                          void *ws, size_t ws_bytes, void *stream) {
    int rc = check_sizes("mtp_linear", dtype, rows, in, out, offsets, n_sets);
    if (rc != MTP_OK) return rc;
    MTP_REQUIRE(act >= LIN_NONE && act <= LIN_SILU, "mtp_linear: unknown activation %d", act);
    MTP_REQUIRE(ldx >= in && (residual == nullptr || ldr >= out), "mtp_linear: row distance below the row's length");
    if (rows == 0) return MTP_OK;
    MTP_REQUIRE(x && w && y, "mtp_linear: null pointer");
    const int64_t need = mtp_linear_workspace_bytes(dtype, MTP_LINEAR_FORWARD, rows, in, out, n_sets, x, ldx, w, in);
    if ((int64_t)ws_bytes < need || (need > 0 && ws == nullptr)) {
        mtp_set_error("mtp_linear: workspace of %zu bytes, needs %lld", ws_bytes, (long long)need);
        return MTP_E_WORKSPACE;
    }
    return MTP_BY_TYPE(dtype, forward)(x, rows, in, ldx, w, out, bias, act, residual, ldr, offsets, n_sets, y, pre,
                                       reinterpret_cast<char *>(ws), mtp_stream(stream));
}

extern "C" int mtp_linear_act_grad(int dtype, const void *g, const void *pre, int64_t rows, int out, int act,
                                   const int32_t *offsets, int n_sets, void *dz, int64_t lddz, void *stream) {
    int rc = check_sizes("mtp_linear_act_grad", dtype, rows, 1, out, offsets, n_sets);
    if (rc != MTP_OK) return rc;
    MTP_REQUIRE(act >= LIN_NONE && act <= LIN_SILU, "mtp_linear_act_grad: unknown activation %d", act);
    MTP_REQUIRE(lddz >= out, "mtp_linear_act_grad: row distance below the row's length");
    if (rows == 0) return MTP_OK;
    MTP_REQUIRE(g && pre && dz, "mtp_linear_act_grad: null pointer");
    const int sz = elem_size(dtype);
    const int vec = out % 8 == 0 && lddz % 8 == 0 &&
                    ((uintptr_t)g | (uintptr_t)pre | (uintptr_t)dz) % (8 * sz) == 0;
    hipStream_t s = mtp_stream(stream);
    const dim3 grid(grid_for(vec ? rows * (out / 8) : rows * out));
    if (dtype == MTP_FLOAT)
        hipLaunchKernelGGL(k_linear_act_grad<float>, grid, dim3(256), 0, s, (const float *)g, (const float *)pre, rows, out, act,
                           offsets, n_sets, (float *)dz, lddz, vec);
    else if (dtype == MTP_BFLOAT16)
        hipLaunchKernelGGL(k_linear_act_grad<__bf16>, grid, dim3(256), 0, s, (const __bf16 *)g, (const __bf16 *)pre, rows, out,
                           act, offsets, n_sets, (__bf16 *)dz, lddz, vec);
    else
        hipLaunchKernelGGL(k_linear_act_grad<_Float16>, grid, dim3(256), 0, s, (const _Float16 *)g, (const _Float16 *)pre, rows,
                           out, act, offsets, n_sets, (_Float16 *)dz, lddz, vec);
    MTP_LAUNCH_CHECK();
    return MTP_OK;
}

extern "C" int mtp_linear_mask_rows(int dtype, const void *g, int64_t rows, int out, const int32_t *offsets, int n_sets, void *dst,
                                    void *stream) {
    int rc = check_sizes("mtp_linear_mask_rows", dtype, rows, 1, out, offsets, n_sets);
    if (rc != MTP_OK) return rc;
    if (rows == 0) return MTP_OK;
    MTP_REQUIRE(g && dst && offsets, "mtp_linear_mask_rows: null pointer");
    hipStream_t s = mtp_stream(stream);
    const dim3 grid(grid_for(rows * out));
    if (dtype == MTP_FLOAT)
        hipLaunchKernelGGL(k_linear_mask_rows<float>, grid, dim3(256), 0, s, (const float *)g, rows, out, offsets, n_sets,
                           (float *)dst);
    else  // the other two types are moved as they are
        hipLaunchKernelGGL(k_linear_mask_rows<_Float16>, grid, dim3(256), 0, s, (const _Float16 *)g, rows, out, offsets, n_sets,
                           (_Float16 *)dst);
    MTP_LAUNCH_CHECK();
    return MTP_OK;
}

extern "C" int mtp_linear_grad_input(int dtype, const void *dz, int64_t rows, int out, int64_t lddz, const void *w, int in,
                                     const int32_t *offsets, int n_sets, void *dx, void *ws, size_t ws_bytes, void *stream) {
    int rc = check_sizes("mtp_linear_grad_input", dtype, rows, in, out, offsets, n_sets);
    if (rc != MTP_OK) return rc;
    MTP_REQUIRE(lddz >= out, "mtp_linear_grad_input: row distance below the row's length");
    if (rows == 0) return MTP_OK;
    MTP_REQUIRE(dz && w && dx, "mtp_linear_grad_input: null pointer");
    const int64_t need = mtp_linear_workspace_bytes(dtype, MTP_LINEAR_GRAD_INPUT, rows, in, out, n_sets, dz, lddz, w, in);
    if ((int64_t)ws_bytes < need || (need > 0 && ws == nullptr)) {
        mtp_set_error("mtp_linear_grad_input: workspace of %zu bytes, needs %lld", ws_bytes, (long long)need);
        return MTP_E_WORKSPACE;
    }
    return MTP_BY_TYPE(dtype, grad_input)(dz, rows, out, lddz, w, in, offsets, n_sets, dx, reinterpret_cast<char *>(ws),
                                          mtp_stream(stream));
}

extern "C" int mtp_linear_grad_weight(int dtype, const void *dz, int64_t rows, int out, int64_t lddz, const void *x, int in,
                                      int64_t ldx, const int32_t *offsets, int n_sets, void *dw, void *db, void *ws,
                                      size_t ws_bytes, void *stream) {
    int rc = check_sizes("mtp_linear_grad_weight", dtype, rows, in, out, offsets, n_sets);
    if (rc != MTP_OK) return rc;
    MTP_REQUIRE(lddz >= out && ldx >= in, "mtp_linear_grad_weight: row distance below the row's length");
    MTP_REQUIRE(dw && (rows == 0 || (dz && x)), "mtp_linear_grad_weight: null pointer");
    const int64_t need = mtp_linear_workspace_bytes(dtype, MTP_LINEAR_GRAD_WEIGHT, rows, in, out, n_sets, dz, lddz, x, ldx);
    if ((int64_t)ws_bytes < need || (need > 0 && ws == nullptr)) {
        mtp_set_error("mtp_linear_grad_weight: workspace of %zu bytes, needs %lld", ws_bytes, (long long)need);
        return MTP_E_WORKSPACE;
    }
    return MTP_BY_TYPE(dtype, grad_weight)(dz, rows, out, lddz, x, in, ldx, offsets, n_sets, dw, db,
                                           reinterpret_cast<char *>(ws), mtp_stream(stream));
}

extern "C" int64_t mtp_linear_backward_workspace_bytes(int dtype, int64_t rows, int in, int out, int n_sets, int act, const void *g,
                                                       const void *w, const void *x, int64_t ldx, int want_x, int want_w) {
    if (rows < 0 || in < 1 || out < 1 || n_sets < 1) return 0;
    return plan_backward(dtype, rows, in, out, n_sets, act, g, w, x, ldx, want_x != 0, want_w != 0).total();
}

extern "C" int mtp_linear_backward(int dtype, const void *g, const void *pre, int act, const void *x, int64_t rows, int in,
                                   int64_t ldx, const void *w, int out, const int32_t *offsets, int n_sets, void *dx, void *dw,
                                   void *db, void *ws, size_t ws_bytes, void *stream) {
    int rc = check_sizes("mtp_linear_backward", dtype, rows, in, out, offsets, n_sets);
    if (rc != MTP_OK) return rc;
    MTP_REQUIRE(dx || dw, "mtp_linear_backward: nothing is asked for");
    MTP_REQUIRE(db == nullptr || dw != nullptr, "mtp_linear_backward: the bias' gradient comes with the weight's");
    const BackwardPlan p = plan_backward(dtype, rows, in, out, n_sets, act, g, w, x, ldx, dx != nullptr, dw != nullptr);
    if ((int64_t)ws_bytes < p.total() || (p.total() > 0 && ws == nullptr)) {
        mtp_set_error("mtp_linear_backward: workspace of %zu bytes, needs %lld", ws_bytes, (long long)p.total());
        return MTP_E_WORKSPACE;
    }
    char *rest = reinterpret_cast<char *>(ws) + p.dz_bytes;
    const void *dz = g;
    if (act != LIN_NONE) {
        rc = mtp_linear_act_grad(dtype, g, pre, rows, out, act, offsets, n_sets, ws, p.lddz, stream);
        if (rc != MTP_OK) return rc;
        dz = ws;
    }
    if (dx != nullptr) {
        rc = mtp_linear_grad_input(dtype, dz, rows, out, p.lddz, w, in, offsets, n_sets, dx, rest, (size_t)p.input_bytes, stream);
        if (rc != MTP_OK) return rc;
    }
    if (dw != nullptr)
        rc = mtp_linear_grad_weight(dtype, dz, rows, out, p.lddz, x, in, ldx, offsets, n_sets, dw, db, rest, (size_t)p.weight_bytes,
                                    stream);
    return rc;
}
