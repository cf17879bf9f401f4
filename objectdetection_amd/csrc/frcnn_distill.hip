// Distillation of the class logits from a teacher's stored top logits, forward and backward.
//
// Row r with teacher logits t_j at labels i_j (j < k; an entry whose label is outside [0, V) or whose
// logit is -inf is not there) and student logits z_v (v < V), temperature T:
//     p = softmax(t / T) over the entries that are there,   q = softmax(z / T) over all V,
//     loss = w T^2 sum_j p_j (log p_j - log q_(i_j)),   d loss / d z_v = w T (q_v - sum_j p_j [i_j = v]).
// A row with w = 0 or no entry takes no part: its loss, lse and gradient are 0 and its logits are not read.
//
// All sums are float32, taken relative to the row's maximum; log q is kept as (z - max)/T - log(sum), so
// the two large terms of z - lse never cancel.  The gradient is written as q first and the few listed
// labels are written again with their p subtracted; a label listed twice gets both.
#include "frcnn_common.h"

namespace frcnn {

constexpr int DS_MAX_K = 1024;

struct DsArgs {
    const void* z; long long ldz;        // [rows,V]
    const void* t;                       // [rows,k]
    const int64_t* idx;                  // [rows,k]
    const float* weight;                 // [rows] or null
    const float* d_loss;                 // [rows] or null: the backward's upstream gradient
    const float* lse_in;                 // [rows]: the backward's
    float scale;                         // factor of the gradient when d_loss is null
    float temperature;
    long long rows; int V, k;
    float* loss; float* lse; void* grad; long long ldg;
};

template <int BLOCK>
__device__ __forceinline__ float ds_block_max(float v, float* sh) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    if constexpr (BLOCK > 64) {
        __syncthreads();
        if (lane_id() == 0) sh[wave_id()] = v;
        __syncthreads();
        v = sh[0];
        for (int w = 1; w < BLOCK / 64; ++w) v = fmaxf(v, sh[w]);
    }
    return v;
}
template <int BLOCK>
__device__ __forceinline__ float ds_block_sum(float v, float* sh) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    if constexpr (BLOCK > 64) {
        __syncthreads();
        if (lane_id() == 0) sh[wave_id()] = v;
        __syncthreads();
        v = sh[0];
        for (int w = 1; w < BLOCK / 64; ++w) v += sh[w];
    }
    return v;
}

constexpr float DS_LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float ds_exp(float x) { return __builtin_amdgcn_exp2f(x * DS_LOG2E); }

// One workgroup per row.  FORWARD: maximum, sum, loss, lse and (grad given) the gradient; else the
// gradient alone, from the forward's lse.
template <typename T, typename U, bool FORWARD, int BLOCK>
__global__ void __launch_bounds__(BLOCK)
distill_row_kernel(DsArgs a) {
    __shared__ float sh[BLOCK / 64 + 1];
    __shared__ float tp[DS_MAX_K];                   // the teacher's entries: t / T, then p
    __shared__ int ti[DS_MAX_K];
    const int tid = threadIdx.x;
    const long long row = blockIdx.x;
    const T* z = (const T*)a.z + row * a.ldz;
    T* grad = a.grad ? (T*)a.grad + row * a.ldg : nullptr;
    const float w = a.weight ? a.weight[row] : 1.0f;
    const float inv_t = 1.0f / a.temperature;

    float tm = -__builtin_inff();
    bool nan_seen = false;
    if (w != 0.f) {
        for (int j = tid; j < a.k; j += BLOCK) {
            const int64_t i = a.idx[row * a.k + j];
            const float t = (float)((const U*)a.t)[row * a.k + j] * inv_t;
            const bool there = i >= 0 && i < a.V && !(t == -__builtin_inff());
            ti[j] = there ? (int)i : -1;
            tp[j] = t;
            if (there) { tm = fmaxf(tm, t); nan_seen |= t != t; }
        }
        tm = ds_block_max<BLOCK>(tm, sh);
        nan_seen = __syncthreads_or(nan_seen);
    }
    if (w == 0.f || (tm == -__builtin_inff() && !nan_seen)) {
        if (FORWARD && tid == 0) { a.loss[row] = 0.f; a.lse[row] = 0.f; }
        if (grad) for (int v = tid; v < a.V; v += BLOCK) grad[v] = (T)0.f;
        return;
    }
    float ts = 0.f;
    for (int j = tid; j < a.k; j += BLOCK)
        if (ti[j] >= 0) ts += ds_exp(tp[j] - tm);
    ts = ds_block_sum<BLOCK>(ts, sh);
    const float log_ts = logf(ts);

    float m, log_s;                                  // log q_v = z_v / T - m - log_s
    if constexpr (FORWARD) {
        m = -__builtin_inff();
        for (int v = tid; v < a.V; v += BLOCK) m = fmaxf(m, (float)z[v] * inv_t);
        m = ds_block_max<BLOCK>(m, sh);
        float s = 0.f;
        for (int v = tid; v < a.V; v += BLOCK) s += ds_exp((float)z[v] * inv_t - m);
        s = ds_block_sum<BLOCK>(s, sh);
        log_s = logf(s);
        float l = 0.f;
        for (int j = tid; j < a.k; j += BLOCK) {
            if (ti[j] < 0) continue;
            const float log_p = tp[j] - tm - log_ts, p = ds_exp(log_p);
            const float log_q = (float)z[ti[j]] * inv_t - m - log_s;
            if (!(p == 0.f)) l += p * (log_p - log_q);
        }
        l = ds_block_sum<BLOCK>(l, sh);
        if (tid == 0) {
            a.loss[row] = w * (a.temperature * a.temperature) * l;
            a.lse[row] = m + log_s;
        }
    } else {
        m = a.lse_in[row];
        log_s = 0.f;
    }
    if (!grad) return;
    const float c = w * a.temperature * (a.d_loss ? a.d_loss[row] : a.scale);
    for (int v = tid; v < a.V; v += BLOCK) grad[v] = (T)(c * ds_exp((float)z[v] * inv_t - m - log_s));
    __syncthreads();
    for (int j = tid; j < a.k; j += BLOCK) {
        const int i = ti[j];
        if (i < 0) continue;
        bool first = true;
        float p = 0.f;
        for (int n = 0; n < a.k; ++n) {
            if (ti[n] != i) continue;
            if (n < j) { first = false; break; }
            p += ds_exp(tp[n] - tm - log_ts);
        }
        if (first) grad[i] = (T)(c * (ds_exp((float)z[i] * inv_t - m - log_s) - p));
    }
}

template <typename T, typename U, bool FORWARD>
static int ds_launch(const DsArgs& a, hipStream_t s) {
    if (a.rows > 0x7FFFFFFFll) return FRCNN_E_UNSUPPORTED;
    FRCNN_LAUNCH((distill_row_kernel<T, U, FORWARD, 256>), dim3((unsigned)a.rows), dim3(256), 0, s, a);
    return FRCNN_OK;
}

template <bool FORWARD>
static int ds_dispatch(const DsArgs& a, int dtype, int t_dtype, hipStream_t s) {
    if (dtype == FRCNN_DT_F32) return ds_launch<float, float, FORWARD>(a, s);
    if (dtype == FRCNN_DT_F16)
        return t_dtype == FRCNN_DT_F32 ? ds_launch<_Float16, float, FORWARD>(a, s)
                                       : ds_launch<_Float16, _Float16, FORWARD>(a, s);
    return t_dtype == FRCNN_DT_F32 ? ds_launch<__bf16, float, FORWARD>(a, s)
                                   : ds_launch<__bf16, __bf16, FORWARD>(a, s);
}

static int ds_check(const void* z, int64_t ldz, int dtype, const void* t, int t_dtype, const int64_t* idx,
                    int64_t rows, int V, int k, float temperature) {
    if (rows < 0 || V <= 0 || k <= 0 || ldz < V) return FRCNN_E_BADARG;
    if (dtype != FRCNN_DT_F32 && dtype != FRCNN_DT_F16 && dtype != FRCNN_DT_BF16) return FRCNN_E_BADARG;
    if (t_dtype != dtype && t_dtype != FRCNN_DT_F32) return FRCNN_E_BADARG;
    if (!(temperature > 0.f) || temperature > 3.0e38f) return FRCNN_E_BADARG;
    if (k > DS_MAX_K || V > 0x40000000) return FRCNN_E_UNSUPPORTED;
    if (rows == 0) return FRCNN_OK;
    if (!z || !t || !idx) return FRCNN_E_BADARG;
    const uintptr_t a = dtype == FRCNN_DT_F32 ? 4 : 2, b = t_dtype == FRCNN_DT_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(z) % a || reinterpret_cast<uintptr_t>(t) % b ||
        reinterpret_cast<uintptr_t>(idx) % 8)
        return FRCNN_E_BADARG;
    return FRCNN_OK;
}

}  // namespace frcnn

using namespace frcnn;

extern "C" int frcnn_distill_loss(const void* logits, int64_t ldz, int dtype, const void* top_values, int t_dtype,
                                  const int64_t* top_index, const float* weight, int64_t rows, int V, int k,
                                  float temperature, float grad_scale, float* loss, float* lse, void* d_logits,
                                  int64_t ldg, frcnn_stream_t stream) {
    const int rc = ds_check(logits, ldz, dtype, top_values, t_dtype, top_index, rows, V, k, temperature);
    if (rc != FRCNN_OK || rows == 0) return rc;
    if (!loss || !lse || (d_logits && ldg < V)) return FRCNN_E_BADARG;
    DsArgs a{};
    a.z = logits; a.ldz = ldz; a.t = top_values; a.idx = top_index; a.weight = weight; a.scale = grad_scale;
    a.temperature = temperature; a.rows = rows; a.V = V; a.k = k;
    a.loss = loss; a.lse = lse; a.grad = d_logits; a.ldg = ldg;
    return ds_dispatch<true>(a, dtype, t_dtype, (hipStream_t)stream);
}

extern "C" int frcnn_distill_bwd(const float* d_loss, const void* logits, int64_t ldz, int dtype,
                                 const void* top_values, int t_dtype, const int64_t* top_index, const float* lse,
                                 const float* weight, int64_t rows, int V, int k, float temperature, void* d_logits,
                                 int64_t ldg, frcnn_stream_t stream) {
    const int rc = ds_check(logits, ldz, dtype, top_values, t_dtype, top_index, rows, V, k, temperature);
    if (rc != FRCNN_OK || rows == 0) return rc;
    if (!d_loss || !lse || !d_logits || ldg < V) return FRCNN_E_BADARG;
    DsArgs a{};
    a.z = logits; a.ldz = ldz; a.t = top_values; a.idx = top_index; a.weight = weight; a.d_loss = d_loss;
    a.lse_in = lse; a.temperature = temperature; a.rows = rows; a.V = V; a.k = k;
    a.grad = d_logits; a.ldg = ldg;
    return ds_dispatch<false>(a, dtype, t_dtype, (hipStream_t)stream);
}
