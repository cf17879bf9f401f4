// Dense layer of the head on 16-bit inputs: out = act(x W + b) + residual with its gradients, on the
// matrix cores (the layers behind the RoI pool, Faster_RCNN/module/model.py:31-38, in f16 / bf16).
//
// All three products (forward, d_x = dz W^T, d_weight = x^T dz) are one kernel
//     D[i][j] = sum_k A[i][k] B[j][k]
// whose operands are read as they lie in memory: either k is the contiguous dimension (x in the
// forward) or the outer one is (both operands of d_weight, a Keras-layout W in the forward); no
// operand is transposed in memory first.  A k-contiguous tile sits in LDS as [outer][64 k] and is
// read 16 bytes per lane; an outer-contiguous tile sits as [64 k][outer] and is read with the
// transposing LDS read (ds_read_b64_tr_b16: 16 lanes give four k rows of 16 values, each gets one
// column of four).  Both are swizzled in 16- / 32-byte pieces so that the reads spread over the
// 64 banks.
//
// v_mfma_f32_16x16x32: products of 16-bit values are exact in float32, the sum over k is float32;
// with the reduction split over workgroups the partial sums are float32 in the workspace and are
// added in slice order, so a call always gives the same bits.  The epilogue works on the float32
// sums: each output is rounded once.
#include "frcnn_common.h"

namespace frcnn {

typedef float dn_f32x4 __attribute__((ext_vector_type(4)));
typedef short dn_s16x4 __attribute__((ext_vector_type(4)));
typedef short dn_s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 dn_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 dn_f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) dn_s16x4 dn_lds_s16x4;

constexpr int DN_BK = 64;                       // k per LDS tile
constexpr int DN_TARGET_WG = 256;               // compute units

__device__ __forceinline__ dn_f32x4 dn_mfma(dn_s16x8 a, dn_s16x8 b, dn_f32x4 c, __bf16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(dn_bf16x8, a),
                                                   __builtin_bit_cast(dn_bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ dn_f32x4 dn_mfma(dn_s16x8 a, dn_s16x8 b, dn_f32x4 c, _Float16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(dn_f16x8, a),
                                                  __builtin_bit_cast(dn_f16x8, b), c, 0, 0, 0);
}

// ---- activations ---------------------------------------------------------------------------------
// Phi(-u) e^(u^2/2) for u >= 0 is smooth and falls like 1/u: a polynomial of degree 8 in
// t = 1 / (1 + 0.33 u) without a constant term, least squares on the relative error over [0, 1e4]
// (1.0e-6; 1.3e-6 evaluated in float32).  The tails keep their relative accuracy because Phi(z) for
// z < 0 is this product itself, not a difference from 1.
struct DnNormal { float cdf, pdf; };
__device__ __forceinline__ DnNormal dn_normal(float z) {
    const float u = fabsf(z);
    const float e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448f);       // e^(-z^2/2)
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.33f, u, 1.0f));
    float q = 0.033283453434705734f;
    q = __builtin_fmaf(q, t, -0.10565749555826187f);
    q = __builtin_fmaf(q, t, 0.06742144376039505f);
    q = __builtin_fmaf(q, t, 0.03343537449836731f);
    q = __builtin_fmaf(q, t, 0.091002456843853f);
    q = __builtin_fmaf(q, t, 0.11721723526716232f);
    q = __builtin_fmaf(q, t, 0.13164693117141724f);
    q = __builtin_fmaf(q, t, 0.13165108859539032f);
    const float tail = q * t * e;
    return {z > 0.f ? 1.0f - tail : tail, e * 0.3989422804014327f};
}
__device__ __forceinline__ float dn_sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));
}
__device__ __forceinline__ float dn_act(float z, int act) {
    if (act == FRCNN_ACT_RELU) return z <= 0.f ? 0.f : z;                     // NaN stays
    if (act == FRCNN_ACT_GELU) return z * dn_normal(z).cdf;
    if (act == FRCNN_ACT_SILU) return z * dn_sigmoid(z);
    return z;
}
// d_out * act'(z); the ReLU's gradient is a selection (0 where z <= 0 or NaN, whatever d_out is)
__device__ __forceinline__ float dn_act_grad(float d, float z, int act) {
    if (act == FRCNN_ACT_RELU) return z > 0.f ? d : 0.f;
    if (act == FRCNN_ACT_GELU) {
        const DnNormal n = dn_normal(z);
        return d * __builtin_fmaf(z, n.pdf, n.cdf);
    }
    if (act == FRCNN_ACT_SILU) {
        const float s = dn_sigmoid(z);
        return d * (s * __builtin_fmaf(z, 1.0f - s, 1.0f));
    }
    return d;
}

// ---- loads and stores of a few neighbouring values, the last of a row guarded -----------------------
// (16- and 8-byte global accesses need no alignment on this machine)
template <typename T>
__device__ __forceinline__ dn_s16x8 dn_load8(const T* p, int valid) {
    dn_s16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
    if (valid >= 8) {
        __builtin_memcpy(&v, p, 16);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < valid) v[e] = __builtin_bit_cast(short, p[e]);
    }
    return v;
}
template <typename T, int W>
__device__ __forceinline__ void dn_load(const T* p, int valid, float* v) {
    T t[W];
    if (valid >= W) {
        __builtin_memcpy(t, p, W * sizeof(T));
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] = (float)t[e];
    } else {
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] = e < valid ? (float)p[e] : 0.f;
    }
}
template <typename T, int W>
__device__ __forceinline__ void dn_store(T* p, int valid, const float* v) {
    T t[W];
#pragma unroll
    for (int e = 0; e < W; ++e) t[e] = (T)v[e];                               // one rounding, to nearest
    if (valid >= W) {
        __builtin_memcpy(p, t, W * sizeof(T));
    } else {
#pragma unroll
        for (int e = 0; e < W; ++e)
            if (e < valid) p[e] = t[e];
    }
}

// ---- the product's arguments -------------------------------------------------------------------------
struct DnEpilogue {
    const void* bias;         // [N'] or null
    const void* residual;     // [M',N'] or null
    void* pre;                // [M',N'] or null
    void* out;                // [M',N'], T or float32
    long long ldr, ldp, ldo;
    int act, out_f32;
};
struct DnGemm {
    const void *a, *b;
    long long lda, ldb, I, J, K;
    long long k_slice;        // k per slice, a multiple of DN_BK
    int splits, tiles_i, tiles_j;
    float* partial;           // [splits][I][Jp], Jp = J rounded up to 4, when splits > 1
    DnEpilogue e;
};

// four neighbouring outputs of one row
template <typename T>
__device__ __forceinline__ void dn_epilogue4(const DnEpilogue& e, long long i, long long j, int valid, dn_f32x4 acc) {
    float v[4] = {acc[0], acc[1], acc[2], acc[3]};
    if (e.bias) {
        float b[4];
        dn_load<T, 4>((const T*)e.bias + j, valid, b);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += b[r];
    }
    if (e.pre) dn_store<T, 4>((T*)e.pre + i * e.ldp + j, valid, v);
    if (e.act != FRCNN_ACT_NONE) {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = dn_act(v[r], e.act);
    }
    if (e.residual) {
        float b[4];
        dn_load<T, 4>((const T*)e.residual + i * e.ldr + j, valid, b);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += b[r];
    }
    if (e.out_f32) dn_store<float, 4>((float*)e.out + i * e.ldo + j, valid, v);
    else dn_store<T, 4>((T*)e.out + i * e.ldo + j, valid, v);
}

// ---- LDS tiles -------------------------------------------------------------------------------------
// position (in 16-byte pieces) of piece `c` of row `r`; its own inverse in c
template <bool KC, int R>
__device__ __forceinline__ int dn_swizzle(int r, int c) {
    if constexpr (KC) return c ^ (r & 7);                                     // [R][8 pieces of 8 k]
    constexpr int m = R >= 128 ? 7 : R / 16 - 1;                              // [64][R / 8 pieces]
    return c ^ ((((r & 3) | ((r >> 1) & 4)) & m) << 1);
}

// One operand's tile, `outer0 ..` by `k0 ..`, from memory into registers (zeros outside) and on into LDS.
template <typename T, bool KC, int R, int NT>
struct DnStage {
    static constexpr int NP = R * 8 / NT;       // 16-byte pieces per thread
    dn_s16x8 v[NP];
    __device__ __forceinline__ void load(const T* p, long long ld, long long outer0, long long outer_end,
                                         long long k0, long long k_end) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int idx = (int)threadIdx.x + NT * i;
            if constexpr (KC) {
                const long long o = outer0 + idx / 8, k = k0 + 8 * (idx % 8);
                const long long left = o < outer_end ? k_end - k : 0;
                v[i] = dn_load8(p + o * ld + k, left > 8 ? 8 : (int)left);
            } else {
                const long long k = k0 + idx / (R / 8), o = outer0 + 8 * (idx % (R / 8));
                const long long left = k < k_end ? outer_end - o : 0;
                v[i] = dn_load8(p + k * ld + o, left > 8 ? 8 : (int)left);
            }
        }
    }
    __device__ __forceinline__ void store(dn_s16x8* lds) const {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int idx = (int)threadIdx.x + NT * i;
            constexpr int P = KC ? 8 : R / 8;
            const int r = idx / P, c = idx % P;
            lds[r * P + dn_swizzle<KC, R>(r, c)] = v[i];
        }
    }
};

// fragment of outer rows o0 .. o0 + 15 (o0 a multiple of 16), k = 32 kk .. 32 kk + 31: lane l holds
// row l % 16, k 8 (l / 16) .. + 7
template <bool KC, int R>
__device__ __forceinline__ dn_s16x8 dn_fragment(const dn_s16x8* lds, int o0, int kk) {
    const int lane = lane_id(), g = lane >> 4, l = lane & 15;
    if constexpr (KC) {
        const int r = o0 + l;
        return lds[r * 8 + dn_swizzle<true, R>(r, kk * 4 + g)];
    } else {
        const int k = kk * 32 + g * 8 + (l >> 2), c = o0 / 8 + ((l & 3) >> 1);
        const short* base = reinterpret_cast<const short*>(lds);
        const short* p0 = base + (k * (R / 8) + dn_swizzle<false, R>(k, c)) * 8 + (l & 1) * 4;
        const short* p1 = base + ((k + 4) * (R / 8) + dn_swizzle<false, R>(k + 4, c)) * 8 + (l & 1) * 4;
        const dn_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((dn_lds_s16x4*)p0);
        const dn_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((dn_lds_s16x4*)p1);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// workgroup id -> tile: every XCD (id % 8) gets a contiguous run of tiles, and a run walks groups of
// eight tile rows column by column, so that the tiles resident on an XCD share A and B panels in its L2
__device__ __forceinline__ void dn_tile(const DnGemm& p, int& ti, int& tj, int& slice) {
    const int n = (int)gridDim.x, id = (int)blockIdx.x, xcd = id & 7, q = n >> 3, r = n & 7;
    int t = xcd * q + (xcd < r ? xcd : r) + (id >> 3);
    const int per = p.tiles_i * p.tiles_j;
    slice = t / per;
    t -= slice * per;
    const int group = 8 * p.tiles_j, g = t / group, first = g * 8;
    const int rows = p.tiles_i - first < 8 ? p.tiles_i - first : 8;
    ti = first + (t - g * group) % rows;
    tj = (t - g * group) / rows;
}

// WI x WJ waves, each (BI / WI) x (BJ / WJ) outputs.  The MFMA's rows are j and its columns i, so that
// a lane ends with four neighbouring outputs of one row.
template <typename T, bool AKC, bool BKC, int BI, int BJ, int WI, int WJ>
__global__ void __launch_bounds__(64 * WI * WJ)
dense_gemm_kernel(DnGemm p) {
    constexpr int NT = 64 * WI * WJ, FI = BI / WI / 16, FJ = BJ / WJ / 16;
    __shared__ dn_s16x8 lds_a[BI * 8], lds_b[BJ * 8];
    int ti, tj, slice;
    dn_tile(p, ti, tj, slice);
    const long long i0 = (long long)ti * BI, j0 = (long long)tj * BJ;
    const long long k0 = slice * p.k_slice;
    const long long k_end = k0 + p.k_slice < p.K ? k0 + p.k_slice : p.K;
    const int wave = wave_id(), wi = (wave / WJ) * (BI / WI), wj = (wave % WJ) * (BJ / WJ);

    dn_f32x4 acc[FI][FJ];
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j) acc[i][j] = dn_f32x4{0.f, 0.f, 0.f, 0.f};

    DnStage<T, AKC, BI, NT> sa;
    DnStage<T, BKC, BJ, NT> sb;
    sa.load((const T*)p.a, p.lda, i0, p.I, k0, k_end);
    sb.load((const T*)p.b, p.ldb, j0, p.J, k0, k_end);
#pragma unroll 1
    for (long long k = k0; k < k_end; k += DN_BK) {
        sa.store(lds_a);
        sb.store(lds_b);
        __syncthreads();
        if (k + DN_BK < k_end) {
            sa.load((const T*)p.a, p.lda, i0, p.I, k + DN_BK, k_end);
            sb.load((const T*)p.b, p.ldb, j0, p.J, k + DN_BK, k_end);
        }
#pragma unroll
        for (int kk = 0; kk < DN_BK / 32; ++kk) {
            dn_s16x8 fa[FI], fb[FJ];
#pragma unroll
            for (int i = 0; i < FI; ++i) fa[i] = dn_fragment<AKC, BI>(lds_a, wi + 16 * i, kk);
#pragma unroll
            for (int j = 0; j < FJ; ++j) fb[j] = dn_fragment<BKC, BJ>(lds_b, wj + 16 * j, kk);
#pragma unroll
            for (int i = 0; i < FI; ++i)
#pragma unroll
                for (int j = 0; j < FJ; ++j) acc[i][j] = dn_mfma(fb[j], fa[i], acc[i][j], T());
        }
        __syncthreads();
    }

    const int lane = lane_id();
    const long long Jp = (p.J + 3) / 4 * 4;
#pragma unroll
    for (int i = 0; i < FI; ++i) {
        const long long gi = i0 + wi + 16 * i + (lane & 15);
        if (gi >= p.I) continue;
#pragma unroll
        for (int j = 0; j < FJ; ++j) {
            const long long gj = j0 + wj + 16 * j + 4 * (lane >> 4);
            const long long left = p.J - gj;
            if (left <= 0) continue;
            if (p.partial)      // columns J .. Jp-1 hold zeros: the operand's tile is zero there
                *reinterpret_cast<dn_f32x4*>(p.partial + (slice * p.I + gi) * Jp + gj) = acc[i][j];
            else
                dn_epilogue4<T>(p.e, gi, gj, left > 4 ? 4 : (int)left, acc[i][j]);
        }
    }
}

// sums of a split product's slices, in slice order, and the epilogue; four outputs per thread
template <typename T>
__global__ void __launch_bounds__(256)
dense_join_kernel(const float* __restrict__ partial, int splits, long long I, long long J, DnEpilogue e) {
    const long long q = (J + 3) / 4, id = (long long)blockIdx.x * 256 + threadIdx.x;
    if (id >= I * q) return;
    const long long i = id / q, j = (id - i * q) * 4, stride = I * q * 4;
    dn_f32x4 v = *reinterpret_cast<const dn_f32x4*>(partial + id * 4);
    for (int s = 1; s < splits; ++s) {
        const dn_f32x4 w = *reinterpret_cast<const dn_f32x4*>(partial + s * stride + id * 4);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += w[r];
    }
    const long long left = J - j;
    dn_epilogue4<T>(e, i, j, left > 4 ? 4 : (int)left, v);
}

// ---- dz = d_out * act'(pre), and column sums per block of rows ----------------------------------------
// A workgroup takes `rows` rows of 8 * CG columns; a thread 8 neighbouring columns of every (256 / CG)-th
// row.  dz (may be null) has rows of ldz elements, a multiple of 8; its columns N .. ldz-1 become 0.
template <typename T, typename D>
__global__ void __launch_bounds__(256)
dense_dz_kernel(const D* __restrict__ d_out, long long ldd, const T* __restrict__ pre, long long ldp, long long M,
                int N, int act, int rows, int cg, T* __restrict__ dz, long long ldz, float* __restrict__ sums) {
    __shared__ float part[256][9];
    const int tid = threadIdx.x, c = tid % cg, rl = tid / cg, rn = 256 / cg;
    const long long col = ((long long)blockIdx.y * cg + c) * 8, r0 = (long long)blockIdx.x * rows;
    const long long r1 = r0 + rows < M ? r0 + rows : M;
    const int valid = N - col > 8 ? 8 : (int)(N - col);
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (valid > 0) {
        for (long long r = r0 + rl; r < r1; r += rn) {
            float d[8];
            dn_load<D, 8>(d_out + r * ldd + col, valid, d);
            if (act != FRCNN_ACT_NONE) {
                float z[8];
                dn_load<T, 8>(pre + r * ldp + col, valid, z);
#pragma unroll
                for (int e = 0; e < 8; ++e) d[e] = e < valid ? dn_act_grad(d[e], z[e], act) : 0.f;
            }
            if (dz) dn_store<T, 8>(dz + r * ldz + col, 8, d);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += d[e];
        }
    }
    if (!sums) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) part[tid][e] = s[e];
    __syncthreads();
    if (rl == 0 && valid > 0) {
        for (int r = 1; r < rn; ++r)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += part[r * cg + c][e];
        for (int e = 0; e < valid; ++e) sums[(long long)blockIdx.x * N + col + e] = s[e];
    }
}

// column sums of `blocks` rows of float32 partial sums: 64 columns per workgroup, 4 threads each
template <typename T>
__global__ void __launch_bounds__(256)
dense_bias_grad_kernel(const float* __restrict__ sums, int blocks, int N, T* __restrict__ d_bias) {
    __shared__ float part[4][64];
    const int c = threadIdx.x & 63, q = threadIdx.x >> 6;
    const int col = blockIdx.x * 64 + c;
    float s = 0.f;
    if (col < N)
        for (int b = q; b < blocks; b += 4) s += sums[(long long)b * N + col];
    part[q][c] = s;
    __syncthreads();
    if (q == 0 && col < N) d_bias[col] = (T)(part[0][c] + part[1][c] + part[2][c] + part[3][c]);
}

template <typename T>
__global__ void __launch_bounds__(256) dense_zero_kernel(T* p, long long rows, long long cols, long long ld) {
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    if (id < rows * cols) p[id / cols * ld + id % cols] = (T)0.f;
}

// ---- host ------------------------------------------------------------------------------------------
struct DnPlan { int bi, bj, splits; long long k_slice, tiles_i, tiles_j; size_t partial_bytes; };

static DnPlan dn_plan(long long I, long long J, long long K) {
    DnPlan p{};
    p.bi = p.bj = 128;
    p.tiles_i = (I + p.bi - 1) / p.bi;
    p.tiles_j = (J + p.bj - 1) / p.bj;
    const long long tiles = p.tiles_i * p.tiles_j, steps = (K + DN_BK - 1) / DN_BK;
    long long splits = tiles >= DN_TARGET_WG ? 1 : 2 * DN_TARGET_WG / tiles;
    if (splits > steps / 4) splits = steps / 4;        // four k steps per slice at least
    if (splits > 32) splits = 32;
    if (splits < 1) splits = 1;
    const long long per = (steps + splits - 1) / splits;
    p.k_slice = per * DN_BK;
    p.splits = (int)((steps + per - 1) / per);         // no empty slice
    if (p.splits < 1) p.splits = 1;
    p.partial_bytes = p.splits > 1 ? (size_t)p.splits * (size_t)I * (size_t)((J + 3) / 4 * 4) * 4 : 0;
    return p;
}

template <typename T, bool AKC, bool BKC>
static int dn_launch_gemm(const DnPlan& pl, const DnGemm& g, hipStream_t stream) {
    const long long blocks = pl.tiles_i * pl.tiles_j * pl.splits;
    if (blocks > 0x7FFFFFFFll) return FRCNN_E_UNSUPPORTED;
    FRCNN_LAUNCH((dense_gemm_kernel<T, AKC, BKC, 128, 128, 2, 2>), dim3((unsigned)blocks), dim3(256), 0, stream, g);
    return FRCNN_OK;
}

template <typename T>
static int dn_product(const void* a, long long lda, bool akc, const void* b, long long ldb, bool bkc, long long I,
                      long long J, long long K, const DnEpilogue& e, void* ws, hipStream_t stream) {
    const DnPlan pl = dn_plan(I, J, K);
    DnGemm g{};
    g.a = a; g.b = b; g.lda = lda; g.ldb = ldb; g.I = I; g.J = J; g.K = K;
    g.k_slice = pl.k_slice; g.splits = pl.splits;
    if (pl.tiles_i > 0x7FFFFF || pl.tiles_j > 0x7FFFFF) return FRCNN_E_UNSUPPORTED;
    g.tiles_i = (int)pl.tiles_i; g.tiles_j = (int)pl.tiles_j;
    g.partial = pl.splits > 1 ? (float*)ws : nullptr;
    g.e = e;
    int rc;
    if (akc && bkc) rc = dn_launch_gemm<T, true, true>(pl, g, stream);
    else if (akc) rc = dn_launch_gemm<T, true, false>(pl, g, stream);
    else rc = dn_launch_gemm<T, false, false>(pl, g, stream);
    if (rc != FRCNN_OK || pl.splits == 1) return rc;
    const long long groups = (I * ((J + 3) / 4) + 255) / 256;
    if (groups > 0x7FFFFFFFll) return FRCNN_E_UNSUPPORTED;
    FRCNN_LAUNCH(dense_join_kernel<T>, dim3((unsigned)groups), dim3(256), 0, stream, (const float*)ws, pl.splits, I,
                 J, e);
    return FRCNN_OK;
}

static size_t dn_up(size_t b) { return (b + 255) / 256 * 256; }

// the backward's workspace: dz, its column sums, then the partial sums of one product at a time
struct DnBwdPlan { bool copy; long long ldz; int rows; long long blocks; size_t dz_bytes, sum_bytes, partial_bytes; };

static DnBwdPlan dn_bwd_plan(long long M, int K, int N, int act, int d_dtype, int dtype, bool aligned) {
    DnBwdPlan p{};
    if (M == 0) return p;                              // nothing to multiply: zeros are stored
    p.copy = act != FRCNN_ACT_NONE || d_dtype != dtype || !aligned;
    p.ldz = (N + 7) / 8 * 8;
    p.rows = 64;
    p.blocks = (M + p.rows - 1) / p.rows;
    if (p.blocks > 4096) {                             // long batches: up to 4,096 partial sums per column
        p.rows = (int)(((M + 4095) / 4096 + 63) / 64 * 64);
        p.blocks = (M + p.rows - 1) / p.rows;
    }
    p.dz_bytes = p.copy ? dn_up((size_t)M * (size_t)p.ldz * 2) : 0;
    p.sum_bytes = dn_up((size_t)p.blocks * (size_t)N * 4);
    const size_t x = dn_plan(M, K, N).partial_bytes, w = dn_plan(K, N, M).partial_bytes;
    const size_t wt = dn_plan(N, K, M).partial_bytes;
    p.partial_bytes = dn_up(x > w ? (x > wt ? x : wt) : (w > wt ? w : wt));
    return p;
}

static bool dn_sizes(int64_t M, int K, int N) { return M >= 0 && M <= (1ll << 40) && K > 0 && N > 0; }
static bool dn_16bit(int dtype) { return dtype == FRCNN_DT_F16 || dtype == FRCNN_DT_BF16; }
static bool dn_even(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

template <typename T>
static int dn_zero(void* p, long long rows, long long cols, long long ld, hipStream_t s) {
    const long long groups = (rows * cols + 255) / 256;
    if (groups > 0x7FFFFFFFll) return FRCNN_E_UNSUPPORTED;
    FRCNN_LAUNCH(dense_zero_kernel<T>, dim3((unsigned)groups), dim3(256), 0, s, (T*)p, rows, cols, ld);
    return FRCNN_OK;
}

template <typename T, typename D>
static int dn_launch_dz(const void* d_out, long long ldd, const void* pre, long long ldp, long long M, int N, int act,
                        const DnBwdPlan& p, void* dz, float* sums, hipStream_t s) {
    const int pieces = (N + 7) / 8;
    int cg = 1;
    while (cg < 32 && cg < pieces) cg *= 2;
    const long long gy = (pieces + cg - 1) / cg;
    if (p.blocks > 0x7FFFFFFFll || gy > 65535) return FRCNN_E_UNSUPPORTED;
    FRCNN_LAUNCH((dense_dz_kernel<T, D>), dim3((unsigned)p.blocks, (unsigned)gy), dim3(256), 0, s, (const D*)d_out,
                 ldd, (const T*)pre, ldp, M, N, act, p.rows, cg, (T*)dz, p.ldz, sums);
    return FRCNN_OK;
}

template <typename T>
static int dn_backward(const void* d_out, long long ldd, int d_dtype, const void* x, long long ldx, const void* w,
                       long long ldw, int w_layout, const void* pre, long long ldp, long long M, int K, int N,
                       int dtype, int act, void* d_x, long long lddx, void* d_w, long long lddw, void* d_bias,
                       char* ws, const DnBwdPlan& p, hipStream_t s) {
    const bool kn = w_layout == FRCNN_W_KN;
    int rc = FRCNN_OK;
    if (M == 0) {
        if (d_w) rc = kn ? dn_zero<T>(d_w, K, N, lddw, s) : dn_zero<T>(d_w, N, K, lddw, s);
        if (rc == FRCNN_OK && d_bias) rc = dn_zero<T>(d_bias, 1, N, N, s);
        return rc;
    }
    void* dz = p.copy ? ws : nullptr;
    float* sums = d_bias ? reinterpret_cast<float*>(ws + p.dz_bytes) : nullptr;
    void* partial = ws + p.dz_bytes + p.sum_bytes;
    if (sums || (dz && (d_x || d_w))) {
        rc = d_dtype == FRCNN_DT_F32 ? dn_launch_dz<T, float>(d_out, ldd, pre, ldp, M, N, act, p, dz, sums, s)
                                     : dn_launch_dz<T, T>(d_out, ldd, pre, ldp, M, N, act, p, dz, sums, s);
        if (rc != FRCNN_OK) return rc;
    }
    if (sums)
        FRCNN_LAUNCH(dense_bias_grad_kernel<T>, dim3((unsigned)((N + 63) / 64)), dim3(256), 0, s, sums,
                     (int)p.blocks, N, (T*)d_bias);
    const void* z = dz ? dz : d_out;
    const long long ldz = dz ? p.ldz : ldd;
    DnEpilogue e{};
    if (d_x) {
        e.out = d_x; e.ldo = lddx;
        rc = dn_product<T>(z, ldz, true, w, ldw, kn, M, K, N, e, partial, s);
        if (rc != FRCNN_OK) return rc;
    }
    if (d_w) {
        e.out = d_w; e.ldo = lddw;
        rc = kn ? dn_product<T>(x, ldx, false, z, ldz, false, K, N, M, e, partial, s)
                : dn_product<T>(z, ldz, false, x, ldx, false, N, K, M, e, partial, s);
    }
    return rc;
}

}  // namespace frcnn

using namespace frcnn;

extern "C" size_t frcnn_dense_fwd_workspace_bytes(int64_t M, int K, int N) {
    if (!dn_sizes(M, K, N) || M == 0) return 0;
    return dn_plan(M, N, K).partial_bytes;
}

extern "C" int frcnn_dense_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, int w_layout, const void* bias,
                               const void* residual, int64_t ldr, int64_t M, int K, int N, int dtype, int act,
                               void* out, int64_t ldo, int out_dtype, void* pre, int64_t ldp, void* workspace,
                               size_t workspace_bytes, frcnn_stream_t stream) {
    if (!dn_sizes(M, K, N) || !dn_16bit(dtype) || (out_dtype != dtype && out_dtype != FRCNN_DT_F32))
        return FRCNN_E_BADARG;
    if (act < FRCNN_ACT_NONE || act > FRCNN_ACT_SILU || (w_layout != FRCNN_W_KN && w_layout != FRCNN_W_NK))
        return FRCNN_E_BADARG;
    if (M == 0) return FRCNN_OK;
    const bool kn = w_layout == FRCNN_W_KN;
    if (!x || !w || !out || ldx < K || ldw < (kn ? N : K) || ldo < N) return FRCNN_E_BADARG;
    if ((residual && ldr < N) || (pre && ldp < N)) return FRCNN_E_BADARG;
    if (!dn_even(x, 2) || !dn_even(w, 2) || !dn_even(bias, 2) || !dn_even(residual, 2) || !dn_even(pre, 2) ||
        !dn_even(out, out_dtype == FRCNN_DT_F32 ? 4 : 2))
        return FRCNN_E_BADARG;
    const size_t need = frcnn_dense_fwd_workspace_bytes(M, K, N);
    if (need && (!workspace || workspace_bytes < need || !dn_even(workspace, 16))) return FRCNN_E_WORKSPACE;
    DnEpilogue e{};
    e.bias = bias; e.residual = residual; e.pre = pre; e.out = out;
    e.ldr = ldr; e.ldp = ldp; e.ldo = ldo; e.act = act; e.out_f32 = out_dtype == FRCNN_DT_F32;
    return dtype == FRCNN_DT_BF16
               ? dn_product<__bf16>(x, ldx, true, w, ldw, !kn, M, N, K, e, workspace, (hipStream_t)stream)
               : dn_product<_Float16>(x, ldx, true, w, ldw, !kn, M, N, K, e, workspace, (hipStream_t)stream);
}

extern "C" size_t frcnn_dense_bwd_workspace_bytes(int64_t M, int K, int N) {
    if (!dn_sizes(M, K, N) || M == 0) return 0;
    const DnBwdPlan p = dn_bwd_plan(M, K, N, FRCNN_ACT_RELU, FRCNN_DT_F32, FRCNN_DT_F16, false);
    return p.dz_bytes + p.sum_bytes + p.partial_bytes;
}

extern "C" int frcnn_dense_bwd(const void* d_out, int64_t ldd, int d_dtype, const void* x, int64_t ldx, const void* w,
                               int64_t ldw, int w_layout, const void* pre, int64_t ldp, int64_t M, int K, int N,
                               int dtype, int act, void* d_x, int64_t lddx, void* d_w, int64_t lddw, void* d_bias,
                               void* workspace, size_t workspace_bytes, frcnn_stream_t stream) {
    if (!dn_sizes(M, K, N) || !dn_16bit(dtype) || (d_dtype != dtype && d_dtype != FRCNN_DT_F32))
        return FRCNN_E_BADARG;
    if (act < FRCNN_ACT_NONE || act > FRCNN_ACT_SILU || (w_layout != FRCNN_W_KN && w_layout != FRCNN_W_NK))
        return FRCNN_E_BADARG;
    const bool kn = w_layout == FRCNN_W_KN;
    if (!d_x && !d_w && !d_bias) return FRCNN_E_BADARG;
    if (d_w && lddw < (kn ? N : K)) return FRCNN_E_BADARG;
    if (!dn_even(d_out, d_dtype == FRCNN_DT_F32 ? 4 : 2) || !dn_even(x, 2) || !dn_even(w, 2) || !dn_even(pre, 2) ||
        !dn_even(d_x, 2) || !dn_even(d_w, 2) || !dn_even(d_bias, 2))
        return FRCNN_E_BADARG;
    if (M > 0) {
        if (!d_out || ldd < N) return FRCNN_E_BADARG;
        if (act != FRCNN_ACT_NONE && (!pre || ldp < N)) return FRCNN_E_BADARG;
        if (d_x && (!w || ldw < (kn ? N : K) || lddx < K)) return FRCNN_E_BADARG;
        if (d_w && (!x || ldx < K)) return FRCNN_E_BADARG;
        const size_t need = frcnn_dense_bwd_workspace_bytes(M, K, N);
        if (!workspace || workspace_bytes < need || !dn_even(workspace, 16)) return FRCNN_E_WORKSPACE;
    }
    const bool aligned = ldd % 8 == 0 && dn_even(d_out, 16);
    const DnBwdPlan p = dn_bwd_plan(M, K, N, act, d_dtype, dtype, aligned);
    return dtype == FRCNN_DT_BF16
               ? dn_backward<__bf16>(d_out, ldd, d_dtype, x, ldx, w, ldw, w_layout, pre, ldp, M, K, N, dtype, act,
                                     d_x, lddx, d_w, lddw, d_bias, (char*)workspace, p, (hipStream_t)stream)
               : dn_backward<_Float16>(d_out, ldd, d_dtype, x, ldx, w, ldw, w_layout, pre, ldp, M, K, N, dtype, act,
                                       d_x, lddx, d_w, lddw, d_bias, (char*)workspace, p, (hipStream_t)stream);
}
