/*
 * The norm at a block's exit, its gate, the scaled residual and the norm at the next block's entry in one pass
 * (ace_block_norm_forward); the entry points of both passes (the backward kernels are in layer_norm_back.hip).
 *
 * Bound by memory: forward reads x and block and writes r and y, nothing else of a row's size moves.  A row belongs to
 * one workgroup with about as many lanes as it has vectors of eight elements (16- and 32-byte accesses) and stays in registers
 * from its first load to its last store.  A workgroup asks for its next row before it computes the one it has, and everything
 * that it reads in between, parameters and the wavefronts' sums, comes from LDS: loads from memory return in order, and a
 * parameter read behind the next row would wait for it.
 *
 * Variance is the mean of squared differences from the mean, in two sums over the row, so that neither a large mean nor a
 * channel far from the others costs digits.
 *
 * 8 x 2,048 rows of 5,120 elements of bfloat16, both norms: 138 us, 4.9 TB/s (a large copy: 5.2); one row of 2,048: 3 us, of a call's
 * 11 (the host's part of it).
 */
#include "layer_norm.h"

namespace {

thread_local hipError_t last_error = hipSuccess;

enum { W2, B2, GATE, W1, B1, PARAMS };

/* mean (0 without `layer`) and 1 / sqrt(variance + eps) of a row; its lanes hold zero past its end */
template <int NV, bool EVEN> __device__ inline float2 norm_of(const f32x8 *u, const int *n, bool layer, float inv, float eps, NormExchange &lds, int &slot) {
    float mean = 0.0f, s = 0.0f;
    if (layer) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) s += u[k][i];
        mean = sum_all(s, lds, slot ^= 1) * inv;
        s = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = (EVEN ? n[k] > 0 : i < n[k]) ? u[k][i] - mean : 0.0f;
            s += d * d;
        }
    return {mean, rsqrtf(sum_all(s, lds, slot ^= 1) * inv + eps)};
}

template <class T, int CAP, int NV, bool EVEN, bool HAS_F, bool ENTRY> __global__ void __launch_bounds__(CAP) norm_forward(const NormArgs a) {
    __shared__ NormExchange lds;
    extern __shared__ f32x4 room[];
    constexpr bool AHEAD = norm_params_in_lds<NV>();
    const int C = a.width;
    uint32_t at[NV];
    int n[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) at[k] = (k * blockDim.x + threadIdx.x) * 8, n[k] = C - (int)at[k];
    const bool exit_norm = a.w2;
    const float inv = 1.0f / C;
    int slot = 0;
    packed8<T> x[NV], f[NV];
    auto ask = [&](int64_t of) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            x[k] = row_load<T, EVEN>(row_at<T>(a.x, of, C), C, at[k], n[k]);
            if (HAS_F) f[k] = row_load<T, EVEN>(row_at<T>(a.f, of, C), C, at[k], n[k]);
        }
    };
#pragma unroll
    for (int k = 0; k < NV; ++k) x[k] = f[k] = 0;
    NormParams<T, NV, EVEN> params = {(T *)room, (int)blockDim.x * NV * 8, C};
    params.put(W2, a.w2, at, n, 1.0f), params.put(B2, a.b2, at, n, 0.0f), params.put(W1, a.w1, at, n, 1.0f), params.put(B1, a.b1, at, n, 0.0f);
    int64_t row = blockIdx.x, gate_row = 0, gate_end = a.rows_per_gate;
    if (row < a.rows) {
        gate_row = row / a.rows_per_gate, gate_end = (gate_row + 1) * a.rows_per_gate;
        params.put(GATE, a.gate ? (const T *)a.gate + gate_row * C : nullptr, at, n, 1.0f);
        if (AHEAD) ask(row);
    }
    for (; row < a.rows; row += gridDim.x) {
        if (row >= gate_end) {
            gate_row = row / a.rows_per_gate, gate_end = (gate_row + 1) * a.rows_per_gate;
            params.put(GATE, (const T *)a.gate + gate_row * C, at, n, 1.0f);
        }
        f32x8 r[NV], z[NV];
        if (!AHEAD) ask(row);
#pragma unroll
        for (int k = 0; k < NV; ++k) r[k] = open8<T>(x[k]), z[k] = open8<T>(f[k]);
        if (AHEAD && row + gridDim.x < a.rows) ask(row + gridDim.x);
        f32x4 st = {0.0f, 1.0f, 0.0f, 1.0f};
        if (HAS_F) {
            if (exit_norm) {
                const float2 m = norm_of<NV, EVEN>(z, n, a.layer, inv, a.eps, lds, slot);
                st.x = m.x, st.y = m.y;
            }
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                z[k] = (z[k] - st.x) * st.y * params.get(W2, a.w2, at[k], n[k], 1.0f) + params.get(B2, a.b2, at[k], n[k], 0.0f);
                const f32x8 by = params.get(GATE, a.gate ? (const T *)a.gate + gate_row * C : nullptr, at[k], n[k], 1.0f);
                r[k] = a.alpha * r[k] + by * z[k];   /* (zero past the row's end: so are the parameters) */
                row_store<T, EVEN>(row_at<T>(a.r, row, C), C, at[k], pack8<T>(r[k]), n[k]);
            }
        }
        if (ENTRY) {
            const float2 m = norm_of<NV, EVEN>(r, n, a.layer, inv, a.eps, lds, slot);
            st.z = m.x, st.w = m.y;
#pragma unroll
            for (int k = 0; k < NV; ++k)
                row_store<T, EVEN>(row_at<T>(a.y, row, C), C, at[k],
                                   pack8<T>((r[k] - m.x) * m.y * params.get(W1, a.w1, at[k], n[k], 1.0f) + params.get(B1, a.b1, at[k], n[k], 0.0f)), n[k]);
        }
        if (threadIdx.x == 0) ((f32x4 *)a.stats)[row] = st;
    }
}

int64_t least(int64_t a, int64_t b) { return a < b ? a : b; }

/* Workgroups that walk over the rows, each with its parameters in LDS: as many as a CU holds at once by their LDS, with 1,536 lanes or
 * fewer.  16,384 rows of bfloat16, up to 1,024, 1,536 and 2,048 lanes and one workgroup per row: 2,048 elements in 51.6, 50.0, 55.7 and
 * 57.2 us; 5,120 in 165, 138, 141 and 177 us.  12,288 elements, of which LDS holds the parameters once: 292 us, with two workgroups 297. */
int64_t grid_of(const NormShape &shape, int64_t rows, int lds) {
    const int64_t by_lanes = shape.lanes > 768 ? 1 : 1536 / shape.lanes;
    return least(rows, 256 * (lds > 0 ? least(by_lanes, 160 * 1024 / lds) : by_lanes));
}

template <class T, int CAP, int NV, bool EVEN, bool HAS_F, bool ENTRY> int launch(const NormArgs &a, const NormShape &shape, hipStream_t stream) {
    const auto kernel = norm_forward<T, CAP, NV, EVEN, HAS_F, ENTRY>;
    static std::atomic<uint64_t> done;
    const int ready = norm_params_in_lds<NV>() ? layer_allow_lds((const void *)kernel, 155 * 1024, done) : ACE_OK;
    if (ready != ACE_OK) return ready;
    const int room = norm_params_in_lds<NV>() ? PARAMS * norm_pitch(shape) * (int)sizeof(T) : 0;
    kernel<<<(uint32_t)grid_of(shape, a.rows, room), shape.lanes, room, stream>>>(a);
    return layer_launched();
}

template <class T> int forward(const NormArgs &a, hipStream_t stream) {
    int rc = ACE_OK;
#define CALL(CAP, NV, EVEN)                                                                                       \
    {                                                                                                             \
        if (!a.f) rc = launch<T, CAP, NV, EVEN, false, true>(a, shape, stream);                             \
        else if (!a.w1) rc = launch<T, CAP, NV, EVEN, true, false>(a, shape, stream);                       \
        else rc = launch<T, CAP, NV, EVEN, true, true>(a, shape, stream);                                   \
    }
    NORM_FOR_SHAPE(CALL, true)
#undef CALL
    return rc;
}

/* Runs of consecutive rows of the backward pass, one per workgroup: as many as the CUs hold at once, as far as lanes with 168
 * registers go.  16,384 rows of bfloat16 in 256, 512 and 1,024 runs: 1,024 elements (128 lanes) in 104, 70 and 61 us; 2,048 in 120, 96 and
 * 100; 4,096 in 178, 178 and 196; 5,120 (640 lanes) in 214, 225 and 225; 12,288 in 528, 553 and 553.  8,144 rows of 1,024 of float32, whose
 * partial sums are no larger than those of bfloat16: 58, 51.7 and 52.9. */
int64_t runs_of(const ace_block_norm_t *a) {
    const int lanes = norm_shape(a->width, a->dtype == ACE_T_F32 ? 4 : 2, false).lanes;
    const int64_t most = lanes > 512 ? 256 : lanes > 128 || a->dtype == ACE_T_F32 ? 512 : 1024;
    const int64_t run = (a->rows + most - 1) / most;
    return (a->rows + run - 1) / run;
}

int64_t gates_of(const ace_block_norm_t *a) { return a->d_gate && a->rows_per_gate < a->rows ? (a->rows + a->rows_per_gate - 1) / a->rows_per_gate : 1; }

bool token_gate(const ace_block_norm_t *a) { return a->d_gate && a->rows_per_gate == 1 && a->rows > 1; }

int check(const ace_block_norm_t *a) {
    if (!a || a->rows < 0 || a->width < 1 || a->dtype < ACE_T_F32 || a->dtype > ACE_T_F16) return ACE_EINVAL;
    if (a->width > ACE_NORM_MAX_WIDTH || a->rows > ((int64_t)1 << 40)) return ACE_ETOOBIG;
    if (a->rows == 0) return ACE_OK;   /* (tensors without elements may have no address) */
    if (!a->d_block && (a->d_gate || a->d_exit_weight)) return ACE_EINVAL;
    if ((a->d_exit_bias && !a->d_exit_weight) || (a->d_entry_bias && !a->d_entry_weight)) return ACE_EINVAL;
    if (!a->d_block && !a->d_entry_weight) return ACE_EINVAL;
    if (a->d_gate && a->rows_per_gate < 1) return ACE_EINVAL;
    if (!a->d_x) return ACE_EINVAL;
    return ACE_OK;
}

NormArgs args_of(const ace_block_norm_t *a) {
    NormArgs k = {};
    k.rows = a->rows, k.rows_per_gate = a->d_gate && a->rows_per_gate <= a->rows ? a->rows_per_gate : a->rows + 1, k.gates = gates_of(a);
    k.width = a->width, k.layer = a->layer, k.alpha = a->d_block ? a->residual_scale : 1.0f, k.eps = a->eps;
    k.x = a->d_x, k.f = a->d_block, k.gate = a->d_gate, k.w2 = a->d_exit_weight, k.b2 = a->d_exit_bias, k.w1 = a->d_entry_weight, k.b1 = a->d_entry_bias;
    return k;
}

}  // namespace

int layer_hip_status(hipError_t e) {
    if (e == hipSuccess) return ACE_OK;
    last_error = e;
    return ACE_EHIP;
}

int layer_allow_lds(const void *kernel, int bytes, std::atomic<uint64_t> &done) {
    int device = 0;
    const int rc = layer_hip_status(hipGetDevice(&device));
    if (rc != ACE_OK) return rc;
    const uint64_t bit = device >= 0 && device < 64 ? (uint64_t)1 << device : 0;
    if (done.load(std::memory_order_acquire) & bit) return ACE_OK;
    if (layer_hip_status(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes)) != ACE_OK) return ACE_EHIP;
    done.fetch_or(bit, std::memory_order_release);
    return ACE_OK;
}

extern "C" int ace_layer_abi_version(void) { return ACE_LAYER_ABI_VERSION; }

extern "C" const char *ace_layer_last_hip_error(void) { return last_error == hipSuccess ? "" : hipGetErrorString(last_error); }

extern "C" const char *ace_layer_strerror(int code) {
    switch (code) {
    case ACE_OK: return "ok";
    case ACE_EINVAL: return "invalid argument";
    case ACE_ETOOBIG: return "larger than the kernels hold";
    case ACE_EHIP: return "HIP error";
    default: return "unknown error";
    }
}

extern "C" int ace_block_norm_forward(const ace_block_norm_t *a, void *d_residual, void *d_normed, float *d_stats, void *stream) {
    const int rc = check(a);
    if (rc != ACE_OK || a->rows == 0) return rc;
    if (!d_stats || (a->d_block && !d_residual) || (a->d_entry_weight && !d_normed)) return ACE_EINVAL;
    NormArgs k = args_of(a);
    k.r = d_residual, k.y = d_normed, k.stats = d_stats;
    const hipStream_t s = (hipStream_t)stream;
    return a->dtype == ACE_T_F32 ? forward<float>(k, s) : a->dtype == ACE_T_BF16 ? forward<bf16>(k, s) : forward<f16>(k, s);
}

extern "C" size_t ace_block_norm_workspace_bytes(const ace_block_norm_t *a) {
    if (check(a) != ACE_OK || a->rows == 0) return 0;
    const int64_t runs = runs_of(a);
    const int64_t rows = (a->d_block ? 2 * (runs + (token_gate(a) ? 0 : gates_of(a) - 1)) : 0) + (a->d_entry_weight ? 2 * runs : 0);
    return (size_t)(rows * a->width) * sizeof(float);
}

extern "C" int ace_block_norm_backward(const ace_block_norm_t *a, const void *g_residual, const void *g_normed, const float *d_stats, void *d_dx,
                                       void *d_dblock, void *d_dgate, void *d_dexit_weight, void *d_dexit_bias, void *d_dentry_weight,
                                       void *d_dentry_bias, void *d_workspace, size_t workspace_bytes, void *stream) {
    const int rc = check(a);
    if (rc != ACE_OK || a->rows == 0) return rc;   /* (the caller clears the sums over no rows) */
    if ((d_dblock && !a->d_block) || (d_dgate && !a->d_gate) || ((d_dexit_weight || d_dexit_bias) && !a->d_exit_weight) ||
        ((d_dentry_weight || d_dentry_bias) && !a->d_entry_weight))
        return ACE_EINVAL;
    if (!d_stats || !d_workspace || workspace_bytes < ace_block_norm_workspace_bytes(a)) return ACE_EINVAL;
    if (gates_of(a) >= (int64_t)65535 * 65535 && d_dgate && !token_gate(a)) return ACE_ETOOBIG;
    NormArgs k = args_of(a);
    k.token_gate = token_gate(a);
    k.runs = runs_of(a), k.run = (a->rows + k.runs - 1) / k.runs;
    k.dr = g_residual, k.dy = g_normed, k.stats = (float *)d_stats;
    k.dx = d_dx, k.df = d_dblock, k.dgate = d_dgate, k.dw2 = d_dexit_weight, k.db2 = d_dexit_bias, k.dw1 = d_dentry_weight, k.db1 = d_dentry_bias;
    const int64_t slots = k.runs + (k.token_gate ? 0 : k.gates - 1);
    float *ws = (float *)d_workspace;
    if (a->d_block) k.sum_a = ws, k.sum_b = ws + slots * a->width, ws += 2 * slots * a->width;
    if (a->d_entry_weight) k.sum_w1 = ws, k.sum_b1 = ws + k.runs * a->width;
    return norm_backward_launch(k, a->dtype, (hipStream_t)stream);
}
