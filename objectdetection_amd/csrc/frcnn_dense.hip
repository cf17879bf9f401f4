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
#include <atomic>
#include <type_traits>

namespace frcnn {

typedef float dn_f32x4 __attribute__((ext_vector_type(4)));
typedef short dn_s16x4 __attribute__((ext_vector_type(4)));
typedef short dn_s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 dn_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 dn_f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) dn_s16x4 dn_lds_s16x4;
typedef __attribute__((address_space(3))) const dn_s16x8 dn_lds_s16x8;

constexpr int DN_CUS = 256;                     // compute units

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
// z < 0 is this product itself, not a difference from 1, and because the exponent z^2 / (2 ln 2) is carried in two
// parts: rounded to one it puts e^(-z^2/2) off by up to 2^-24 of itself, 7e-6 at -12.
struct DnNormal { float cdf, pdf; };
__device__ __forceinline__ DnNormal dn_normal(float z) {
    const float u = fabsf(z);
    const float v = fminf(u, 16.0f), v2 = v * v, c = -0.72134752044448f;     // e^(-z^2/2) is 0 from 14.4 on
    const float h = v2 * c, l = __builtin_fmaf(__builtin_fmaf(v, v, -v2), c, __builtin_fmaf(v2, c, -h) + v2 * -9.6298e-9f);
    float e = __builtin_amdgcn_exp2f(h);
    e = __builtin_fmaf(e, l * 0.69314718f, e);
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

// the first `valid` of eight values, without a branch where all are known to be wanted
template <bool ALL, typename T>
__device__ __forceinline__ void dn_store_some(T* p, int valid, const float (&v)[8]) {
    T t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = (T)v[e];
    if constexpr (ALL) {
        __builtin_memcpy(p, t, 8 * sizeof(T));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
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
    long long outer_a, outer_b;   // I, J rounded up to whole pieces where the operand's rows are that long
    long long k_slice;        // k per slice: an even number of steps
    int splits, tiles_i, tiles_j;
    float* partial;           // [splits][I][Jp], Jp = J rounded up to 4, when splits > 1
    long long low_a, low_b;   // TWO: elements from the operand that is dz to its low part, 0 for the other one
    float low_scale, scale;   // TWO: factors of the low part's product and of the result,
    const float* scale_at;    // the latter in memory where it comes from the values (or null)
    DnEpilogue e;
};

// W neighbouring outputs of one row, `valid` of them inside, from their float32 sums
template <typename T, int W>
__device__ __forceinline__ void dn_epilogue(const DnEpilogue& e, long long i, long long j, int valid, float* v) {
    if (e.bias) {
        float b[W];
        dn_load<T, W>((const T*)e.bias + j, valid, b);
#pragma unroll
        for (int r = 0; r < W; ++r) v[r] += b[r];
    }
    if (e.pre) dn_store<T, W>((T*)e.pre + i * e.ldp + j, valid, v);
    if (e.act != FRCNN_ACT_NONE) {
#pragma unroll
        for (int r = 0; r < W; ++r) v[r] = dn_act(v[r], e.act);
    }
    if (e.residual) {
        float b[W];
        dn_load<T, W>((const T*)e.residual + i * e.ldr + j, valid, b);
#pragma unroll
        for (int r = 0; r < W; ++r) v[r] += b[r];
    }
    if (e.out_f32) dn_store<float, W>((float*)e.out + i * e.ldo + j, valid, v);
    else dn_store<T, W>((T*)e.out + i * e.ldo + j, valid, v);
}

// ---- LDS tiles -------------------------------------------------------------------------------------
// position (in 16-byte pieces) of piece `c` of row `r`; its own inverse in c.  Sixteen lanes that read
// 16 rows of a k-contiguous tile, or four rows of 32 bytes twice in an outer-contiguous one, touch every
// bank once (no conflict counted)
template <bool KC, int R, int BK>
__device__ __forceinline__ int dn_swizzle(int r, int c) {
    if constexpr (KC) return c ^ ((r >> 1) & 7);                              // [R][8 pieces of 8 k]
    else if constexpr (R == 64) return c ^ ((((r >> 1) & 1) | ((r >> 2) & 2)) << 1);      // [BK][8 pieces]
    else return c ^ (((r & 3) | ((r >> 1) & 4)) << 1);                        // [BK][R / 8 pieces]
}

// tile number -> tile: every XCD (number % 8) gets a contiguous run of tiles, and a run walks groups of eight
// tile rows column by column, so that the tiles resident on an XCD share A and B panels in its L2 (groups of
// four or sixteen: within 1 % on most products, 2 % and 12 % slower with W as [N,K])
__device__ __forceinline__ void dn_tile(const DnGemm& p, int id, int n, int& ti, int& tj, int& slice) {
    const int xcd = id & 7, q = n >> 3, r = n & 7;
    int t = xcd * q + (xcd < r ? xcd : r) + (id >> 3);
    const int per = p.tiles_i * p.tiles_j;
    slice = t / per;
    t -= slice * per;
    const int group = 8 * p.tiles_j, g = t / group, first = g * 8;
    const int rows = p.tiles_i - first < 8 ? p.tiles_i - first : 8;
    ti = first + (t - g * group) % rows;
    tj = (t - g * group) / rows;
}

// the thread's number, not known to be the same as before: what is computed from it is computed again where
// it is needed instead of waiting in registers through the products
__device__ __forceinline__ int dn_thread() {
    int t = (int)threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

// A wave's results, (16 FI) x (16 FJ) at (i0, j0): the float32 partial sums of a slice, or the outputs.
// Sixteen rows at a time turn round through LDS (the wave's own dn_turn_bytes), so that a lane holds eight
// neighbouring outputs and the lanes of a row store whole 128-byte lines.  Inside the matrix nothing is
// guarded, the bias is loaded once (a lane's columns stay the same) and the residual of the next sixteen
// rows is on its way before the stores of these: memory operations finish in order, and a load waited for
// behind stores, or a guarded one, costs their whole way to memory (6 us per 256 x 256 tile).
// The turned rows' 16-byte pieces are exchanged by the row number instead of padded: the large tile's ring
// and turns are all of a compute unit's LDS.
template <int FJ> constexpr int dn_turn_bytes() { return 16 * FJ * 64; }

template <typename T, int FI, int FJ, bool FULL>
__device__ __forceinline__ void dn_write_out(const DnGemm& p, const dn_f32x4 (&acc)[FI][FJ], int slice, long long i0,
                                             long long j0, char* turn) {
    constexpr int S = FJ * 64, Q = 2 * FJ, RP = 64 / Q;           // bytes per row, pieces of 8 per row, rows per pass
    constexpr int NP = 16 / RP;                                   // passes per sixteen rows
    const int lane = dn_thread() & 63;
    if (p.partial) {            // columns J .. Jp-1 may be written and are never read as results
        const long long Jp = (p.J + 3) / 4 * 4;
#pragma unroll
        for (int i = 0; i < FI; ++i) {
            const long long gi = i0 + 16 * i + (lane & 15);
            if (gi >= p.I) continue;
#pragma unroll
            for (int j = 0; j < FJ; ++j) {
                const long long gj = j0 + 16 * j + 4 * (lane >> 4);
                if (gj < Jp) *reinterpret_cast<dn_f32x4*>(p.partial + (slice * p.I + gi) * Jp + gj) = acc[i][j];
            }
        }
        return;
    }
    if (j0 >= p.J) return;
    const long long row0 = i0 + lane / Q, gj = j0 + 8 * (lane % Q);
    const int valid = p.J - gj > 8 ? 8 : (int)(p.J - gj);
    constexpr int X = 4 * FJ - 1;                                 // 16-byte pieces per row, less one
    char* put = turn + (lane & 15) * S;
    const char* get = turn + (lane / Q) * S;
    const DnEpilogue& ep = p.e;
    const bool has_res = FULL && ep.residual, has_pre = FULL && ep.pre, f32 = FULL && ep.out_f32;
    // INNER: whole pieces in all lanes; else value by value, loads at clamped places instead of under a guard
    auto body = [&](auto inner) {
        constexpr bool INNER = decltype(inner)::value;
        auto load = [&](const T* row, short (&to)[8]) {
            if constexpr (INNER) {
                __builtin_memcpy(to, row + gj, 16);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const long long j = gj + e < p.J ? gj + e : p.J - 1;
                    __builtin_memcpy(&to[e], row + j, 2);
                }
            }
        };
        auto store = [&](auto* to, const float (&v)[8]) { dn_store_some<INNER>(to, valid, v); };
        float bias[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        short now[NP][8] = {}, next[NP][8] = {};
        auto fetch = [&](int i, short (&to)[NP][8]) {
#pragma unroll
            for (int r = 0; r < NP; ++r) {
                const long long gi = row0 + 16 * i + r * RP;
                load((const T*)ep.residual + (gi < p.I ? gi : p.I - 1) * ep.ldr, to[r]);
            }
        };
        if constexpr (FULL) {
            if (ep.bias) {
                short t[8];
                load((const T*)ep.bias, t);
#pragma unroll
                for (int e = 0; e < 8; ++e) bias[e] = (float)__builtin_bit_cast(T, t[e]);
            }
            if (has_res) fetch(0, now);
        }
        // a loop, not FI copies: code that runs once per workgroup is fetched from beyond the instruction cache
#pragma unroll 1
        for (int i = 0; i < FI; ++i) {
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int c = 0; c < FI; ++c)
                if (i == c) {
                    asm volatile("; rows %0" ::"n"(c));           // keeps the branches apart: acc stays in registers
#pragma unroll
                    for (int j = 0; j < FJ; ++j) {
                        dn_f32x4 a = acc[c][j];
                        asm volatile("" : "+v"(a));
                        *reinterpret_cast<dn_f32x4*>(put + (((4 * j + (lane >> 4)) ^ lane) & X) * 16) = a;
                    }
                }
            __builtin_amdgcn_wave_barrier();
            if (has_res && i + 1 < FI) fetch(i + 1, next);
#pragma unroll
            for (int r = 0; r < NP; ++r) {
                const long long gi = row0 + 16 * i + r * RP;
                const bool inside = gi < p.I;
                float v[8];
                const int row = r * RP + lane / Q;                // of the sixteen
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    __builtin_memcpy(v + 4 * h, get + r * RP * S + (((2 * (lane % Q) + h) ^ row) & X) * 16, 16);
                if constexpr (FULL) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += bias[e];
                    if (has_pre && inside) store((T*)ep.pre + gi * ep.ldp + gj, v);
                    if (ep.act != FRCNN_ACT_NONE) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = dn_act(v[e], ep.act);
                    }
                    if (has_res) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] += (float)__builtin_bit_cast(T, now[r][e]);
                    }
                }
                if (inside) {
                    if (f32) store((float*)ep.out + gi * ep.ldo + gj, v);
                    else store((T*)ep.out + gi * ep.ldo + gj, v);
                }
            }
#pragma unroll
            for (int r = 0; r < NP; ++r)
#pragma unroll
                for (int e = 0; e < 8; ++e) now[r][e] = next[r][e];
        }
    };
    if (j0 + 16 * FJ <= p.J) body(std::true_type());
    else body(std::false_type());
}

// ---- the product -----------------------------------------------------------------------------------------
// Tiles go from memory to LDS directly (global_load_lds, 16 bytes per lane, the swizzle applied to the
// source address because the destination is linear in the lane).  The reduction is walked in steps of 32 k:
// while the fragments of step s, already in registers, are multiplied, those of step s + 1 are read from
// LDS and later ones are in flight, in a ring of RING steps.  An outer-contiguous operand is copied a step at a
// time, at step s that of s + RING; a k-contiguous one two steps at a time (64 k: whole 128-byte lines, copies of
// half lines took L2 twice the requests: 1,282 TFLOP/s at 8,192 cubed, 1,444 this way), at every odd s those of
// s + RING - 1 and s + RING.  A handover says that the copies step s + 1 needs have arrived (the newer ones stay in
// flight) and that every wave has read step s, whose place is then filled again.  Rows outside the
// operand repeat its last row (their results are not stored); k outside reads a page of zeros.
// RING is 4.  With both operands k-contiguous that is one copy of two steps in flight, which the steps of the smaller
// tiles do not cover: there it is 6 where a compute unit holds one workgroup (1,000 x 4,096 x 4,096 54 -> 47 us
// with the same tiles, 2,000 x 4,096 x 4,096 77 -> 60; with more workgroups the room is better used by a second one:
// 50,000 x 64 x 64 6.6 us, 8.2 with 6).  Eight cost another 1.2 us to fill.
// What bounds it: the clock (1.83 GHz under this load) and the matrix cores, busy 74 (W as [N,K]) to 84 % (d_weight of
// 16,000 x 25,088 x 4,096) of its cycles.  8,192 cubed in bf16: 1,430 to 1,450 TFLOP/s with W as [N,K], 1,460 to 1,550
// as Keras kernel, 1,445 to 1,550 for d_weight (from card to card).
constexpr int DN_SK = 32;
__device__ const __attribute__((aligned(16))) uint32_t dn_zeros[4] = {0, 0, 0, 0};

// (m0 is a reserved register: the compiler sets it before each use of its own)
__device__ __forceinline__ void dn_dma(uint32_t lds, const void* base, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :: "s"(lds), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void dn_dma(uint32_t lds, const void* p) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :: "s"(lds), "v"(p) : "memory");
}
// all but the newest N copies of this wave have arrived and its LDS reads are done; then the same of all waves
template <int N>
__device__ __forceinline__ void dn_handover() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <typename T, bool KC, int R, int NT>
struct DnCopy {
    static constexpr int CK = KC ? 2 * DN_SK : DN_SK;             // k per copy
    static constexpr int P = KC ? CK / 8 : R / 8, NP = R * CK / 8 / NT;   // pieces per LDS row, per thread
    static constexpr uint32_t BYTES = R * CK * 2;
    uint32_t off[NP];
    const char* base;          // at (outer0, k)
    long long step;            // bytes per copy
    __device__ __forceinline__ void init(const T* p, long long ld, long long outer0, long long outer_end,
                                         long long k0) {
        const long long ld2 = ld * 2, left = outer_end - outer0;
        const int tid = dn_thread();
        base = reinterpret_cast<const char*>(p) + (KC ? outer0 * ld2 + k0 * 2 : k0 * ld2 + outer0 * 2);
        step = KC ? CK * 2 : CK * ld2;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int idx = tid + NT * i;
            int r = idx / P, c = dn_swizzle<KC, R, CK>(r, idx % P);
            if constexpr (KC) r = r < left ? r : (int)left - 1;
            else c = 8 * c + 8 <= left ? c : (int)(left / 8) - 1;
            off[i] = (uint32_t)r * (uint32_t)ld2 + (uint32_t)c * 16u;
        }
    }
    // the k at `base` to LDS byte address `lds` (of this wave's first piece); base moves on
    __device__ __forceinline__ void issue(uint32_t lds) {
#pragma unroll
        for (int i = 0; i < NP; ++i) dn_dma(lds + (uint32_t)(NT * i * 16), base, off[i]);
        base += step;
    }
    // the same where only the first `valid` k are inside
    __device__ __forceinline__ void issue(uint32_t lds, int valid) {
        if (valid >= CK) return issue(lds);
        const int tid = dn_thread();
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int idx = tid + NT * i, r = idx / P;
            const int k = KC ? 8 * dn_swizzle<KC, R, CK>(r, idx % P) : r;
            dn_dma(lds + (uint32_t)(NT * i * 16), k < valid ? base + off[i] : reinterpret_cast<const char*>(dn_zeros));
        }
        base += step;
    }
};

// A wave's fragments of 16 outer rows from `o0` on, of any step in the ring, from one LDS address per lane:
// fragment f is a constant further where k is contiguous, and at the address with f in its swizzled
// bits where it is not; the place in the ring is a constant offset of the instruction (an operand's ring
// lies within 64 KB, its first byte on a multiple of 2 KB).
template <bool KC, int R, int RING>
struct DnReader {
    uint32_t at;
    __device__ __forceinline__ void init(uint32_t lds, int o0) {
        const int lane = lane_id(), g = lane >> 4, l = lane & 15;
        if constexpr (KC) {
            at = lds + (uint32_t)((o0 + l) * 8 + dn_swizzle<true, R, 64>(l, g)) * 16u;
        } else {
            const int k = g * 8 + (l >> 2);
            at = lds + (uint32_t)(k * (R / 8) + dn_swizzle<false, R, DN_SK>(k, o0 / 8 + ((l & 3) >> 1))) * 16u +
                 (uint32_t)(l & 1) * 8u;
        }
    }
    // keeps the compiler from holding an address per fragment in registers
    __device__ __forceinline__ void renew() { asm volatile("" : "+v"(at)); }
    __device__ __forceinline__ dn_s16x8 read(int f, int step) const {
        const uint32_t ring = (uint32_t)(step % RING);
        if constexpr (KC) {     // the odd step is the second half of the row: pieces 4 .. 7
            const uint32_t a = (at ^ ((ring & 1u) * 64u)) + (ring >> 1) * (R * 128u);
            return *(dn_lds_s16x8*)(uintptr_t)(a + (uint32_t)f * 2048u);
        } else {
            const uint32_t a = (at ^ ((uint32_t)f * 32u)) + ring * (R * 64u);
            const dn_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((dn_lds_s16x4*)(uintptr_t)a);
            const dn_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((dn_lds_s16x4*)(uintptr_t)(a + 8u * R));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// FULL: with bias, pre, activation, residual or a float32 output in the epilogue (the forward).
// STAY: the workgroup takes tile `id` and every `stride`-th after it; the first copies of the next tile leave
// before the results of this one are written, and arrive meanwhile.  `tiles`: tiles and slices in all.
// TWO: the operand that is dz comes as the sum of two values of its type (dense_dz_kernel); the reduction is walked
// twice over the same other operand, the low part first, with the sums in the same registers (d_weight of 16,000 x
// 4,096 x 4,096: 746 us, 1,440 TFLOP/s of the two products).
template <typename T, bool AKC, bool BKC, int BI, int BJ, int WI, int WJ, int RING, bool FULL, bool STAY, bool TWO>
__device__ __forceinline__ void dn_gemm(const DnGemm& p, int tiles, int id, int stride, char* dn_lds) {
    constexpr int NT = 64 * WI * WJ, FI = BI / WI / 16, FJ = BJ / WJ / 16;
    constexpr int READS = FI * (AKC ? 1 : 2) + FJ * (BKC ? 1 : 2);  // LDS reads per wave and step
    constexpr uint32_t RING_A = BI * DN_SK * 2 * RING, RING_B = BJ * DN_SK * 2 * RING;
    const int wave = __builtin_amdgcn_readfirstlane(wave_id());
    const int wi = (wave / WJ) * (BI / WI), wj = (wave % WJ) * (BJ / WJ);
    char* turn = dn_lds + (STAY ? RING_A + RING_B : 0) + wave * dn_turn_bytes<FJ>();

    using CopyA = DnCopy<T, AKC, BI, NT>;
    using CopyB = DnCopy<T, BKC, BJ, NT>;
    // copies per thread: of the operands that are copied every step, of those copied every other step
    constexpr int EVERY = (AKC ? 0 : CopyA::NP) + (BKC ? 0 : CopyB::NP);
    constexpr int OTHER = (AKC ? CopyA::NP : 0) + (BKC ? CopyB::NP : 0);
    // newer ones that a handover before an even / an odd step leaves in flight
    constexpr int EVEN = (RING / 2 - 1) * OTHER + (RING - 2) * EVERY, ODD = EVEN - OTHER;
    CopyA ca;
    CopyB cb;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)dn_lds;
    const uint32_t la = lds0 + (uint32_t)wave * 1024u, lb = la + RING_A;
    DnReader<AKC, BI, RING> qa;
    DnReader<BKC, BJ, RING> qb;
    qa.init(lds0, wi);
    qb.init(lds0 + RING_A, wj);
    auto read = [&](int s, dn_s16x8 (&ra)[FI], dn_s16x8 (&rb)[FJ]) {
        qa.renew();
        qb.renew();
#pragma unroll
        for (int j = 0; j < FJ; ++j) rb[j] = qb.read(j, s);
#pragma unroll
        for (int i = 0; i < FI; ++i) ra[i] = qa.read(i, s);
    };
    long long i0 = 0, j0 = 0, k0 = 0, k_end = 0;
    int slice = 0, n = 0;                              // n: steps
    // the copies for step s: every-step operands (EV), and with an even s every-other-step ones (OT)
    auto issue = [&](int s, bool ev, bool ot) {
        if (s >= n) return;
        const long long left = k_end - k0 - (long long)s * DN_SK;
        const int valid = left < 2 * DN_SK ? (int)left : 2 * DN_SK;
        const uint32_t ring = (uint32_t)(s % RING);
        if (AKC ? ot : ev) ca.issue(la + ring * (BI * 64u), valid);
        if (BKC ? ot : ev) cb.issue(lb + ring * (BJ * 64u), valid);
    };
    auto start = [&](int id) {
        int ti, tj;
        dn_tile(p, id, tiles, ti, tj, slice);
        i0 = (long long)ti * BI;
        j0 = (long long)tj * BJ;
        k0 = slice * p.k_slice;
        k_end = k0 + p.k_slice < p.K ? k0 + p.k_slice : p.K;
        n = (int)((k_end - k0 + DN_SK - 1) / DN_SK);
        ca.init((const T*)p.a + (TWO ? p.low_a : 0), p.lda, i0, AKC ? p.I : p.outer_a, k0);
        cb.init((const T*)p.b + (TWO ? p.low_b : 0), p.ldb, j0, BKC ? p.J : p.outer_b, k0);
#pragma unroll
        for (int s = 0; s < RING; ++s) issue(s, true, s % 2 == 0);
    };

    start(id);
    dn_f32x4 acc[FI][FJ];
    bool low = TWO;                                    // the low part is being multiplied
#pragma unroll 1
    while (true) {
        dn_s16x8 fa[2][FI], fb[2][FJ];
        if (!TWO || low) {
#pragma unroll
            for (int i = 0; i < FI; ++i)
#pragma unroll
                for (int j = 0; j < FJ; ++j) acc[i][j] = dn_f32x4{0.f, 0.f, 0.f, 0.f};
        }
        auto multiply = [&](const dn_s16x8 (&ra)[FI], const dn_s16x8 (&rb)[FJ]) {
#pragma unroll
            for (int i = 0; i < FI; ++i)
#pragma unroll
                for (int j = 0; j < FJ; ++j) acc[i][j] = dn_mfma(rb[j], ra[i], acc[i][j], T());
        };
        // steps 0 and 1 (behind the last tile's results all but the newest are waited for: no harm)
        if (n >= RING) dn_handover<EVEN>();
        else dn_handover<0>();
        read(0, fa[0], fb[0]);
        int s = 0;
        // whole steps, a ring's length at a time so that every LDS address is a constant; no branch inside
#pragma unroll 1
        for (; s + 2 * RING < n; s += RING) {
#pragma unroll
            for (int u = 0; u < RING; ++u) {
                if (u & 1) {
                    dn_handover<ODD>();
                    if (AKC) ca.issue(la + ((u + RING - 1) % RING) * (BI * 64u));
                    if (BKC) cb.issue(lb + ((u + RING - 1) % RING) * (BJ * 64u));
                } else if (EVERY) {
                    dn_handover<EVEN>();
                }
                if (!AKC) ca.issue(la + u * (BI * 64u));
                if (!BKC) cb.issue(lb + u * (BJ * 64u));
                read(u + 1, fa[(u + 1) & 1], fb[(u + 1) & 1]);
                multiply(fa[u & 1], fb[u & 1]);
                // the reads of the next step between the products of this one, early
                __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
#pragma unroll
                for (int q = 0; q < READS; ++q) {
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, FI * FJ, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // the last steps: up to two rings' lengths, the last one maybe cut short
        auto step = [&](const dn_s16x8 (&ra)[FI], const dn_s16x8 (&rb)[FJ], dn_s16x8 (&na)[FI], dn_s16x8 (&nb)[FJ]) {
            if (s + 1 < n) {
                if (s + RING - 1 >= n) dn_handover<0>();
                else if (s & 1) dn_handover<ODD>();
                else dn_handover<EVEN>();
                if (s & 1) issue(s + RING - 1, false, true);
                issue(s + RING, true, false);
                read(s + 1, na, nb);
            }
            multiply(ra, rb);
            ++s;
        };
#pragma unroll 1
        while (s < n) {
            step(fa[0], fb[0], fa[1], fb[1]);
            if (s < n) step(fa[1], fb[1], fa[0], fb[0]);
        }
        dn_handover<0>();                              // every wave has read the last step: the ring is free
        if constexpr (TWO) {
            const float f = low ? p.low_scale : p.scale_at ? *p.scale_at : p.scale;
#pragma unroll
            for (int i = 0; i < FI; ++i)
#pragma unroll
                for (int j = 0; j < FJ; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[i][j][r] *= f;
            __builtin_amdgcn_sched_barrier(0);
            low = !low;
            if (!low) {                                // back to the first step, of the high part
                ca.base -= (AKC ? (n + 1) / 2 : n) * ca.step + 2 * p.low_a;
                cb.base -= (BKC ? (n + 1) / 2 : n) * cb.step + 2 * p.low_b;
#pragma unroll
                for (int s = 0; s < RING; ++s) issue(s, true, s % 2 == 0);
                continue;
            }
        }
        const long long oi = i0 + wi, oj = j0 + wj;
        const int os = slice;
        id += stride;
        const bool more = STAY && id < tiles;
        if (more) start(id);
        dn_write_out<T, FI, FJ, FULL>(p, acc, os, oi, oj, turn);
        if (!more) return;
    }
}

template <typename T, bool AKC, bool BKC, int BI, int BJ, int WI, int WJ, int RING, bool FULL, bool STAY, bool TWO>
__global__ void __launch_bounds__(64 * WI * WJ)
dense_gemm_kernel(DnGemm p, int tiles) {
    extern __shared__ __attribute__((aligned(16))) char dn_lds[];    // A's ring, B's, the turns (STAY)
    dn_gemm<T, AKC, BKC, BI, BJ, WI, WJ, RING, FULL, STAY, TWO>(p, tiles, (int)blockIdx.x, (int)gridDim.x, dn_lds);
}

// ---- few rows ------------------------------------------------------------------------------------------
// Up to 32 rows (I): the product reads B once and little else, so what counts is how soon and how wide the
// loads of B leave.  A workgroup owns 16 (k contiguous) or 32 (outer contiguous) columns and its eight waves
// share out the reduction in pieces of 64 k: a wave's load covers whole 128-byte lines of 16 rows of B, or
// 64-byte pieces of 16 k (neighbouring workgroups on the same XCD share the lines), and three pieces are loaded
// ahead (waiting for the oldest alone takes as long as for the three together).  A fragment of A comes straight
// from memory (every workgroup reads the same few rows: L2).  An outer-contiguous piece is turned round by the
// transposing LDS read in the wave's own LDS.  The eight sums are added in wave order.  The MFMA's k order is free as
// long as both operands agree: lane group g takes k 16 g .. 16 g + 15 of a piece in two instructions (k contiguous),
// or 8 g .. 8 g + 7 of each half.
// One row x 4,096 x 4,096 bf16, W as [N,K]: 8.3 us, 4.0 TB/s; Keras kernel of 4,096 x 84: 8.6 us.  An outer-contiguous B
// of 4,096 rows, read in half lines, comes at half the rate: 17.5 us at 4,096 x 4,096 (what holds it up is not known).
// Both parts of a dz are multiplied against each load of B.
constexpr int DN_FEW = 32, DN_FW = 8, DN_FS = 3;   // most rows; waves; pieces on their way

template <typename T, bool BKC, int MB, bool TWO>
__global__ void __launch_bounds__(64 * DN_FW) dense_few_rows_kernel(DnGemm p) {
    constexpr int JB = BKC ? 1 : 2, NL = BKC ? 2 : 4;             // 16-column blocks; loads of B per piece and lane
    __shared__ dn_f32x4 sums[DN_FW][JB * MB][64];
    __shared__ dn_s16x8 turn[BKC ? 1 : DN_FW][BKC ? 1 : 256];     // [64 k][4 pieces of 8 columns] per wave
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), g = lane >> 4, l = lane & 15;
    // the last columns are the row's last ones: what they share with their neighbour is not stored
    const unsigned xcd = blockIdx.x & 7, per = gridDim.x >> 3, rest = gridDim.x & 7;
    const long long jw = (long long)(!BKC && gridDim.x >= 128 ? xcd * per + (xcd < rest ? xcd : rest) + (blockIdx.x >> 3)
                                                              : blockIdx.x) * (16 * JB);
    const long long j0 = !BKC && jw > p.J - 32 && p.J >= 32 ? p.J - 32 : jw;
    const int slice = blockIdx.y;
    const long long k0 = slice * p.k_slice, k_end = k0 + p.k_slice < p.K ? k0 + p.k_slice : p.K;
    const T* A = (const T*)p.a;
    const T* B = (const T*)p.b;
    const T* rows[MB];
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        const long long i = 16 * m + l;
        rows[m] = A + (i < p.I ? i : p.I - 1) * p.lda;
    }
    const long long jl = j0 + l < p.J ? j0 + l : p.J - 1;         // k contiguous: this lane's row of B
    // Columns outside B are loaded too, from the rows behind, and not stored; the last rows have none behind them.
    const long long whole = BKC || j0 + 16 * JB <= p.J || p.K - 7 > k_end ? k_end : p.K - 7;
    const int last = (int)(p.J - 1 - j0) / 8 * 8, c8 = 8 * (lane & 3) < last ? 8 * (lane & 3) : last;
    const int jv = (int)(p.J - j0 - 8 * (lane & 3) < 8 ? p.J - j0 - 8 * (lane & 3) : 8);

    constexpr int NA = TWO ? 4 : 2;                               // loads of A per row: 2 and 2 of the low part
    dn_s16x8 b[DN_FS][NL], a[DN_FS][MB][NA];
    auto load = [&](long long k, dn_s16x8 (&rb)[NL], dn_s16x8 (&ra)[MB][NA]) {
#pragma unroll
        for (int h = 0; h < NL; ++h) {
            const T* q = BKC ? B + jl * p.ldb + k + 16 * g + 8 * h
                             : B + (k + 16 * h + (lane >> 2)) * p.ldb + j0 + c8;
            __builtin_memcpy(&rb[h], q, 16);
        }
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int h = 0; h < NA; ++h)
                __builtin_memcpy(&ra[m][h], rows[m] + (h < 2 ? 0 : p.low_a) + k +
                                                (BKC ? 16 * g + 8 * (h & 1) : 32 * (h & 1) + 8 * g), 16);
    };
    auto load_some = [&](long long k, dn_s16x8 (&rb)[NL], dn_s16x8 (&ra)[MB][NA]) {
        auto at = [&](const T* q, long long kk) {
            const long long left = k_end - kk;
            return dn_load8(q + kk, left > 8 ? 8 : (int)left);
        };
#pragma unroll
        for (int h = 0; h < NL; ++h) {
            if constexpr (BKC) {
                rb[h] = at(B + jl * p.ldb, k + 16 * g + 8 * h);
            } else {
                const long long kk = k + 16 * h + (lane >> 2);
                rb[h] = dn_load8(B + kk * p.ldb + j0 + 8 * (lane & 3), kk < k_end ? jv : 0);
            }
        }
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int h = 0; h < NA; ++h)
                ra[m][h] = at(rows[m] + (h < 2 ? 0 : p.low_a), k + (BKC ? 16 * g + 8 * (h & 1) : 32 * (h & 1) + 8 * g));
    };
    dn_f32x4 acc[JB][MB], acc_low[JB][MB];
#pragma unroll
    for (int j = 0; j < JB; ++j)
#pragma unroll
        for (int m = 0; m < MB; ++m) acc[j][m] = acc_low[j][m] = dn_f32x4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](dn_s16x8 (&rb)[NL], dn_s16x8 (&ra)[MB][NA]) {
        if constexpr (BKC) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int m = 0; m < MB; ++m) {
                    acc[0][m] = dn_mfma(rb[h], ra[m][h], acc[0][m], T());
                    if constexpr (TWO) acc_low[0][m] = dn_mfma(rb[h], ra[m][2 + h], acc_low[0][m], T());
                }
        } else {
            // row k, 32-byte half c / 2 exchanged where k has bit 3: two lane groups meet no bank twice
            dn_s16x8* lds = turn[wave];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int h = 0; h < NL; ++h) {
                const int k = 16 * h + (lane >> 2), c = lane & 3;
                lds[k * 4 + (c ^ ((k >> 2) & 2))] = rb[h];
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < JB; ++j) {
                    const int k = 32 * h + 8 * g + (l >> 2), c = (2 * j + ((l & 3) >> 1)) ^ ((k >> 2) & 2);
                    const short* q = reinterpret_cast<const short*>(lds) + (k * 4 + c) * 8 + (l & 1) * 4;
                    const dn_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((dn_lds_s16x4*)q);
                    const dn_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((dn_lds_s16x4*)(q + 4 * 32));
                    const dn_s16x8 f = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                    for (int m = 0; m < MB; ++m) {
                        acc[j][m] = dn_mfma(f, ra[m][h], acc[j][m], T());
                        if constexpr (TWO) acc_low[j][m] = dn_mfma(f, ra[m][2 + h], acc_low[j][m], T());
                    }
                }
        }
    };
    constexpr long long STEP = 64 * DN_FW;
    long long k = k0 + 64 * wave;
    const int n = k + 64 <= whole ? (int)((whole - k - 64) / STEP) + 1 : 0;              // whole pieces
#pragma unroll
    for (int u = 0; u < DN_FS; ++u)
        if (u < n) load(k + u * STEP, b[u], a[u]);
    int s = 0;
#pragma unroll 1
    for (; s + 2 * DN_FS <= n; s += DN_FS) {
#pragma unroll
        for (int u = 0; u < DN_FS; ++u) {
            multiply(b[u], a[u]);
            load(k + DN_FS * STEP, b[u], a[u]);
            k += STEP;
        }
    }
#pragma unroll 1
    for (; s < n; s += DN_FS) {
#pragma unroll
        for (int u = 0; u < DN_FS; ++u)
            if (s + u < n) {
                multiply(b[u], a[u]);
                if (s + u + DN_FS < n) load(k + DN_FS * STEP, b[u], a[u]);
                k += STEP;
            }
    }
#pragma unroll 1
    for (; k < k_end; k += STEP) {                     // pieces that are cut short or come last in a narrow B
        load_some(k, b[0], a[0]);
        multiply(b[0], a[0]);
    }
    if constexpr (TWO) {
        const float scale = p.scale_at ? *p.scale_at : p.scale;
#pragma unroll
        for (int j = 0; j < JB; ++j)
#pragma unroll
            for (int m = 0; m < MB; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    acc[j][m][r] = (acc[j][m][r] + acc_low[j][m][r] * p.low_scale) * scale;
    }
#pragma unroll
    for (int j = 0; j < JB; ++j)
#pragma unroll
        for (int m = 0; m < MB; ++m) sums[wave][j * MB + m][lane] = acc[j][m];
    __syncthreads();
    if (wave >= JB * MB) return;
    dn_f32x4 v = sums[0][wave][lane];
#pragma unroll
    for (int w = 1; w < DN_FW; ++w) {
        const dn_f32x4 o = sums[w][wave][lane];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += o[r];
    }
    const long long i = 16 * (wave % MB) + l, j = j0 + 16 * (wave / MB) + 4 * g, left = p.J - j;
    if (i >= p.I || left <= 0 || j + 4 <= jw) return;
    float o[4] = {v[0], v[1], v[2], v[3]};
    if (p.partial) {
        float* to = p.partial + (slice * p.I + i) * ((p.J + 3) / 4 * 4) + j;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (j + r >= jw && r < left) to[r] = o[r];
    } else if (j >= jw) {
        dn_epilogue<T, 4>(p.e, i, j, left > 4 ? 4 : (int)left, o);
    } else {                                           // the first of them belong to the neighbour
#pragma unroll
        for (int r = 1; r < 4; ++r)
            if (j + r >= jw) dn_epilogue<T, 1>(p.e, i, j + r, 1, &o[r]);
    }
}

// a / b for a below 2^40: by 32-bit division where that does (a 64-bit one is a hundred instructions)
__device__ __forceinline__ long long dn_divide(long long a, long long b) {
    return a < 0x80000000ll && b < 0x80000000ll ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}

// sums of a split product's slices, in slice order, and the epilogue; four outputs per thread; of one product
// or two.  Bound by the partial sums' way from memory: eight slices of 128 x 4,096 4.9 us, two of 2,000 x 4,096
// (65.5 MB, 16.4 written) 13.4 us
struct DnJoin { const float* partial; long long I, J, blocks; int splits; DnEpilogue e; };

template <typename T>
__global__ void __launch_bounds__(64) dense_join_kernel(DnJoin one, DnJoin two) {
    const bool first = (long long)blockIdx.x < one.blocks;
    const DnJoin p = first ? one : two;
    const long long q = (p.J + 3) / 4, id = ((long long)blockIdx.x - (first ? 0 : one.blocks)) * 64 + threadIdx.x;
    if (id >= p.I * q) return;
    const long long i = dn_divide(id, q), j = (id - i * q) * 4, stride = p.I * q * 4;
    dn_f32x4 v = *reinterpret_cast<const dn_f32x4*>(p.partial + id * 4);
    int s = 1;
    for (; s + 8 <= p.splits; s += 8) {                // eight slices on their way at once
        dn_f32x4 w[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) w[q] = *reinterpret_cast<const dn_f32x4*>(p.partial + (s + q) * stride + id * 4);
#pragma unroll
        for (int q = 0; q < 8; ++q)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] += w[q][r];
    }
    for (; s < p.splits; ++s) {
        const dn_f32x4 w = *reinterpret_cast<const dn_f32x4*>(p.partial + s * stride + id * 4);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += w[r];
    }
    const long long left = p.J - j;
    float o[4] = {v[0], v[1], v[2], v[3]};
    dn_epilogue<T, 4>(p.e, i, j, left > 4 ? 4 : (int)left, o);
}

// ---- operands whose rows are not whole 16-byte pieces --------------------------------------------------
// are copied once to rows that are, with zeros behind their end: a piece per thread, in one launch for all
// of a call's operands (777 x 1,003 and 1,003 x 531 f16: 4.3 us, latency; 8,192 x 4,099 bf16 22 us, 6.1 TB/s)
struct DnPack { const void* src; void* dst; long long rows, cols, ld, pieces; };   // pieces of 8 per row of dst
struct DnPacks { DnPack of[2]; long long blocks_first, blocks; };                  // workgroups of 256 pieces

template <typename T>
__device__ __forceinline__ void dn_pack_piece(const DnPacks& packs, long long block) {
    const bool first = block < packs.blocks_first;
    const DnPack p = packs.of[first ? 0 : 1];
    const long long id = (block - (first ? 0 : packs.blocks_first)) * 256 + threadIdx.x;
    if (id >= p.rows * p.pieces) return;
    const long long r = dn_divide(id, p.pieces), c = 8 * (id - r * p.pieces), left = p.cols - c;
    const dn_s16x8 v = dn_load8((const T*)p.src + r * p.ld + c, left > 8 ? 8 : (int)left);
    reinterpret_cast<dn_s16x8*>(p.dst)[id] = v;
}
template <typename T>
__global__ void __launch_bounds__(256) dense_pack_kernel(DnPacks packs) {
    dn_pack_piece<T>(packs, blockIdx.x);
}

// ---- dz = d_out * act'(pre) and its column sums ---------------------------------------------------------
// A workgroup takes `rows` rows of 8 * cg columns; a thread 8 neighbouring columns of every (256 / cg)-th
// row.  dz (may be null) has rows of ldz elements, a multiple of 8; its columns N .. ldz-1 become 0.  Where dz is
// no value of the type (GELU, SiLU, a float32 d_out) it is kept as the sum of two that are:
// scale dz = high + low / low_up with high the nearest value and low what is left of it.  That is 2^-16 relative
// in bfloat16 and 2^-22 in float16, for twice the matrix operations; one value (2^-8 and 2^-11) makes the gradients
// 1.4 times as wrong as their own rounding does.  The sums of the unrounded values go to d_bias where one workgroup
// has all rows, else to `sums`, a row per block of rows.  The workgroups behind the first `blocks` pack the products'
// operands.  16,000 x 84 bf16: 7 us; 1,111 x 333 f16 with SiLU, packing 779 x 333 and 1,111 x 779: 9 us (latency both)
struct DnDz {
    const void *d_out, *pre;
    void *dz, *d_bias;
    float* sums;
    long long ldd, ldp, ldz, M, rows, row_blocks, blocks, low;    // low: elements from dz to its low part, or 0
    float scale, low_up;
    const float* most;        // largest |d_out| by the workgroups of dense_most_kernel, or null: `scale` is taken
    float* back;              // where workgroup 0 leaves the inverse of the scale
    int n_most, N, act, cg;
};
// the nearest value of T, and the rest of v times up (0 behind infinities and NaN; a finite v that rounds to an
// infinity leaves the largest finite value and the rest)
template <typename T>
__device__ __forceinline__ void dn_two(float v, float up, float& high, float& low) {
    const float most = std::is_same<T, __bf16>::value ? 3.3895313892515355e38f : 65504.0f;
    high = (float)(T)v;
    if (fabsf(v) < __builtin_inff()) high = fabsf(high) <= most ? high : __builtin_copysignf(most, v);
    low = fabsf(v) < __builtin_inff() ? (v - high) * up : 0.f;
}
// The largest finite |d_out|: a float32 gradient need not lie in float16's range, so for float16 it is brought there by
// a power of two (of the largest value's exponent: 2^14 .. 2^15) that the products take off again.
// At most 256 workgroups, each leaves one value (16,000 x 21: 4.7 us, latency).
__global__ void __launch_bounds__(256) dense_most_kernel(const float* d_out, long long ldd, long long M, int N, float* most) {
    __shared__ float part[4];
    const long long pieces = (N + 7) / 8, step = (long long)gridDim.x * 256;
    float m = 0.f;
    for (long long id = (long long)blockIdx.x * 256 + threadIdx.x; id < M * pieces; id += step) {
        const long long r = dn_divide(id, pieces), c = 8 * (id - r * pieces), left = N - c;
        float d[8];
        dn_load<float, 8>(d_out + r * ldd + c, left > 8 ? 8 : (int)left, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(d[e]) < __builtin_inff() ? fabsf(d[e]) : 0.f);
    }
    for (int d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
    if (lane_id() == 0) part[wave_id()] = m;
    __syncthreads();
    if (threadIdx.x == 0) most[blockIdx.x] = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
}

template <typename T, typename D>
__global__ void __launch_bounds__(256) dense_dz_kernel(DnDz p, DnPacks packs) {
    __shared__ float part[4][32][9], top[4];
    if ((long long)blockIdx.x >= p.blocks) return dn_pack_piece<T>(packs, blockIdx.x - p.blocks);
    float scale = p.scale;
    if (p.most) {
        float m = (int)threadIdx.x < p.n_most ? p.most[threadIdx.x] : 0.f;
        for (int d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
        if (lane_id() == 0) top[wave_id()] = m;
        __syncthreads();
        m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        int e = 14 + 127 - (int)(__float_as_uint(m) >> 23);          // below the normal range as at its end
        e = m == 0.f ? 0 : e < 126 ? e : 126;
        scale = __uint_as_float((unsigned)(127 + e) << 23);
        if (blockIdx.x == 0 && threadIdx.x == 0) *p.back = __uint_as_float((unsigned)(127 - e) << 23);
    }
    const D* d_out = (const D*)p.d_out;
    const T* pre = (const T*)p.pre;
    T* dz = (T*)p.dz;
    const int tid = threadIdx.x, c = tid & (p.cg - 1), rl = tid / p.cg, rn = 256 / p.cg;
    const long long column = dn_divide(blockIdx.x, p.row_blocks), block = blockIdx.x - column * p.row_blocks;
    const long long col = (column * p.cg + c) * 8, r0 = block * p.rows, r1 = r0 + p.rows < p.M ? r0 + p.rows : p.M;
    const int valid = p.N - col > 8 ? 8 : (int)(p.N - col);
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    auto row = [&](long long r, const float (&d)[8], const float (&z)[8]) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < valid ? dn_act_grad(d[e], z[e], p.act) : 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] += v[e];
        if (dz && p.low) {
            float h[8], l[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) dn_two<T>(v[e] * scale, p.low_up, h[e], l[e]);
            dn_store<T, 8>(dz + r * p.ldz + col, 8, h);
            dn_store<T, 8>(dz + p.low + r * p.ldz + col, 8, l);
        } else if (dz) {
            dn_store<T, 8>(dz + r * p.ldz + col, 8, v);
        }
    };
    if (valid > 0) {
        const bool act_any = p.act != FRCNN_ACT_NONE;
        long long r = r0 + rl;
        for (; r + rn < r1; r += 2 * rn) {             // two rows on their way
            float d0[8], d1[8], z0[8] = {}, z1[8] = {};
            dn_load<D, 8>(d_out + r * p.ldd + col, valid, d0);
            dn_load<D, 8>(d_out + (r + rn) * p.ldd + col, valid, d1);
            if (act_any) {
                dn_load<T, 8>(pre + r * p.ldp + col, valid, z0);
                dn_load<T, 8>(pre + (r + rn) * p.ldp + col, valid, z1);
            }
            row(r, d0, z0);
            row(r + rn, d1, z1);
        }
        if (r < r1) {
            float d0[8], z0[8] = {};
            dn_load<D, 8>(d_out + r * p.ldd + col, valid, d0);
            if (act_any) dn_load<T, 8>(pre + r * p.ldp + col, valid, z0);
            row(r, d0, z0);
        }
    }
    if (!p.sums && !p.d_bias) return;
    for (int d = p.cg; d < 64; d *= 2)                 // the wave's lanes of the same columns, then the four waves
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] += __shfl_xor(s[e], d);
    if (lane_id() < p.cg)
#pragma unroll
        for (int e = 0; e < 8; ++e) part[wave_id()][c][e] = s[e];
    __syncthreads();
    if (tid >= p.cg || valid <= 0) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = (part[0][c][e] + part[1][c][e]) + (part[2][c][e] + part[3][c][e]);
    if (p.d_bias) {
        for (int e = 0; e < valid; ++e) ((T*)p.d_bias)[col + e] = (T)s[e];
    } else {
        for (int e = 0; e < valid; ++e) p.sums[block * p.N + col + e] = s[e];
    }
}

// column sums of `blocks` rows of float32 partial sums: 16 columns per workgroup, NT / 16 threads each, four
// rows on their way per thread (16,000 rows of 84: 4 us)
struct DnBiasGrad { const float* sums; void* d_bias; int blocks, N; };

template <typename T, int NT>
__device__ __forceinline__ void dn_bias_grad(const DnBiasGrad& p, int block, float (*part)[17]) {
    const int c = threadIdx.x & 15, q = threadIdx.x >> 4;
    const int col = block * 16 + c;
#pragma unroll
    for (int g = q; g < 64; g += NT / 16) {            // the same 64 sums however many threads there are
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        if (col < p.N)
            for (int b = g; b < p.blocks; b += 256)
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (b + 64 * u < p.blocks) s[u] += p.sums[(long long)(b + 64 * u) * p.N + col];
        part[g][c] = (s[0] + s[1]) + (s[2] + s[3]);
    }
    __syncthreads();
    if (q < 4) {                                       // 16 rows each
        float v = part[16 * q][c];
#pragma unroll
        for (int r = 1; r < 16; ++r) v += part[16 * q + r][c];
        v += __shfl_xor(v, 16);
        v += __shfl_xor(v, 32);
        if (q == 0 && col < p.N) ((T*)p.d_bias)[col] = (T)v;
    }
}
template <typename T>
__global__ void __launch_bounds__(1024) dense_bias_grad_kernel(DnBiasGrad p) {
    __shared__ float part[64][17];
    dn_bias_grad<T, 1024>(p, (int)blockIdx.x, part);
}

// ---- the products of a small backward, and the rest of its bias gradient, in one launch -------------------
// d_x and d_w leave most of the chip idle each, and a launch takes longer on the host than such a product on
// the GPU: workgroups of d_x, then of d_w, then of the bias gradient.
template <typename T, bool BKC, bool TWO>
__global__ void __launch_bounds__(256) dense_pair_kernel(DnGemm x, int tiles_x, DnGemm w, int tiles_w, DnBiasGrad b) {
    extern __shared__ __attribute__((aligned(16))) char dn_lds[];
    const int id = (int)blockIdx.x;
    if (id < tiles_x) dn_gemm<T, true, BKC, 64, 128, 1, 4, BKC ? 6 : 4, false, false, TWO>(x, tiles_x, id, 0, dn_lds);
    else if (id < tiles_x + tiles_w)
        dn_gemm<T, false, false, 64, 128, 1, 4, 4, false, false, TWO>(w, tiles_w, id - tiles_x, 0, dn_lds);
    else dn_bias_grad<T, 256>(b, id - tiles_x - tiles_w, reinterpret_cast<float(*)[17]>(dn_lds));
}

template <typename T>
__global__ void __launch_bounds__(256) dense_zero_kernel(T* p, long long rows, long long cols, long long ld) {
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    if (id < rows * cols) p[id / cols * ld + id % cols] = (T)0.f;
}

// ---- host ------------------------------------------------------------------------------------------
struct DnPlan { int bi, bj, splits; long long k_slice, tiles_i, tiles_j; size_t partial_bytes; };

// Workgroup tiles: what a step of 32 k takes in us per round over the chip, and where one round is all (alone); the
// same with both operands k-contiguous (W as [N,K]); the rest of a workgroup (start, first copies, results) and how many
// are resident.  What follows takes the pair of tile and split with the shortest sum: steps and rounds, or what the
// operands take at 3.81 TB/s and what tiles copy again at 26.2 TB/s (all compute units) if that is longer, plus 0.3 of
// the latter, plus the join of a split.  The constants are fitted to 132 products from 40 x 1,024 x 1,024 to 25,088 x
// 4,096 x 2,000, each measured with every tile and split: what is taken is 1.4 % slower than the best of them in the
// mean.  4,000 x 4,096 x 4,096 wants the large tile (103 us; 119 and 130 from the next two), 2,000 x 25,088 x 4,096 two
// slices of it (307; 330 from 128 x 256 unsplit), 128 x 25,088 x 4,096 eight slices of 128 x 128 (53.5; 55.9 from
// sixteen of 128 x 256), 16,000 x 4,096 x 24 three of them (33; 44.7 from 256 x 256), 1,024 cubed the small tile (9.6;
// 12.5).
struct DnTile { int bi, bj; double step, alone, step_kc, alone_kc, fixed; int resident; };
constexpr DnTile DN_TILES[] = {{256, 256, 0.70, 0.595, 0.77, 0.69, 6.8, 1},
                               {128, 256, 0.388, 0.411, 0.44, 0.38, 4.9, 1},
                               {128, 128, 0.236, 0.28, 0.312, 0.25, 4.3, 2},
                               {64, 128, 0.18, 0.22, 0.153, 0.145, 3.18, 3}};

constexpr long long DN_MAX_LD = 1ll << 21;             // a tile's rows lie within 2 GiB of each other
// a launch has fewer than 2^32 threads
static bool dn_grid(long long blocks, int threads) { return blocks * threads < 1ll << 32; }

// Whether a product of I rows reads its operands as they are.  Large weights of whole pieces are left to the
// tiles: the few rows' kernel reads half lines of an outer-contiguous B (1 x 4,096 x 4,096 as Keras kernel 17.5 us,
// 13.2 by tiles; 1 x 25,088 x 4,096 56 and 39; 1 x 1,024 x 1,024 4.6 and 8.0), and A again for every 16 columns
// (W as [N,K], 32 x 25,088 x 4,096: 78 us, 43 by tiles; 16 x 25,088 x 4,096 54 and 42; 16 x 4,096 x 4,096 10.8 and 13.9).
// Weights from memory, not from the last-level cache, in all of these.
static bool dn_few(long long I, long long J, long long K, bool bkc, bool whole_b) {
    return I <= DN_FEW && !(whole_b && K <= DN_MAX_LD && (bkc ? I : 1) * J * K >= (bkc ? 1ll << 30 : 1ll << 23));
}

// akc: A is k-contiguous (the forward and d_x); only those products have few rows
static DnPlan dn_plan(long long I, long long J, long long K, bool akc, bool bkc, bool few) {
    DnPlan p{};
    if (akc && few) {
        // one workgroup per 16 or 32 columns; a long reduction is split where that leaves compute units idle
        p.bi = 0;
        p.bj = bkc ? 16 : 32;
        p.tiles_i = 1;
        p.tiles_j = (J + p.bj - 1) / p.bj;
        const long long pieces = (K + 64 * DN_FW - 1) / (64 * DN_FW);
        long long splits = pieces >= 16 ? DN_CUS / p.tiles_j : 1;
        if (splits > pieces / 4) splits = pieces / 4;
        if (splits < 1) splits = 1;
        const long long per = (pieces + splits - 1) / splits;
        p.k_slice = per * 64 * DN_FW;
        p.splits = (int)((pieces + per - 1) / per);
        p.partial_bytes = p.splits > 1 ? (size_t)p.splits * (size_t)I * (size_t)((J + 3) / 4 * 4) * 4 : 0;
        return p;
    }
    const long long steps = (K + DN_SK - 1) / DN_SK;
    const double bytes = 2.0 * ((double)I * K + (double)J * K + (double)I * J);
    double best = 0.0;
    for (const DnTile& t : DN_TILES) {
        const long long ti = (I + t.bi - 1) / t.bi, tj = (J + t.bj - 1) / t.bj;
        const double step = bkc && akc ? t.step_kc : t.step, alone = bkc && akc ? t.alone_kc : t.alone;
        for (int want : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
            if (want > 1 && steps < 8 * want) break;       // eight steps per slice at least
            const long long per = ((steps + want - 1) / want + 1) / 2 * 2, splits = (steps + per - 1) / per;
            const double groups = (double)(ti * tj) * (double)splits;
            const double waves = groups <= DN_CUS ? 1.0 : __builtin_ceil(groups / DN_CUS);
            double us = per * (waves > 1.0 ? waves * step : alone) + t.fixed * __builtin_ceil(waves / t.resident);
            // what memory gives, and what L2 gives again
            // (rows outside the operand repeat one row: counted half)
            const double copied = groups * per * ((I < t.bi ? (I + t.bi) / 2 : t.bi) +
                                                  (J < t.bj ? (J + t.bj) / 2 : t.bj)) * (2.0 * DN_SK);
            const double stream = (bytes / 3.81e6 + (copied > bytes ? copied - bytes : 0.0) / 2.62e7) *
                                  (groups < DN_CUS ? DN_CUS / groups : 1.0);
            us = (us < stream ? stream : us) + 0.3 * stream;
            if (splits > 1) us += 2.35 + 0.349 * splits + (double)splits * I * J * 8.0 / 8.92e6;
            if (p.bi && us > best) continue;
            best = us;
            p.bi = t.bi; p.bj = t.bj;
            p.tiles_i = ti; p.tiles_j = tj;
            p.splits = (int)splits; p.k_slice = per * DN_SK;
        }
    }
    p.partial_bytes = p.splits > 1 ? (size_t)p.splits * (size_t)I * (size_t)((J + 3) / 4 * 4) * 4 : 0;
    return p;
}

// lets a kernel use `bytes` of LDS on the current device; said once per kernel and device
static bool dn_raise_lds(const void* kernel, int bytes, std::atomic<uint64_t>& raised) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return false;
    const uint64_t bit = 1ull << (dev & 63);
    if (dev < 64 && (raised.load(std::memory_order_relaxed) & bit)) return true;
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return false;
    raised.fetch_or(bit, std::memory_order_relaxed);
    return true;
}

template <typename T, bool AKC, bool BKC, int BI, int BJ, int WI, int WJ, int RING, bool FULL, bool TWO>
static int dn_launch_kernel(const DnGemm& g, unsigned tiles, hipStream_t stream) {
    // One workgroup of the large tile is all that a compute unit holds: it stays for the tiles of its XCD
    // (16,384 x 64 x 4,096: 32.8 us; 36.5 with a workgroup per tile).  Not with the full epilogue and not where
    // both operands are outer-contiguous: there the next tile's addresses do not fit beside the sums in 256
    // registers, what is parked in memory costs the products 20 %, and computing them again behind the results
    // gains less than 1 %.
    constexpr bool STAY = BI == 256 && BJ == 256 && AKC && !FULL;
    constexpr int lds = RING * (BI + BJ) * DN_SK * 2 + (STAY ? WI * WJ * dn_turn_bytes<BJ / WJ / 16>() : 0);
    static_assert(lds <= 160 * 1024, "LDS of a compute unit");
    const unsigned blocks = STAY && tiles > DN_CUS ? DN_CUS : tiles;
    static std::atomic<uint64_t> raised{0};
    if (!dn_raise_lds(reinterpret_cast<const void*>(dense_gemm_kernel<T, AKC, BKC, BI, BJ, WI, WJ, RING, FULL, STAY, TWO>), lds, raised))
        return FRCNN_E_LAUNCH;
    FRCNN_LAUNCH((dense_gemm_kernel<T, AKC, BKC, BI, BJ, WI, WJ, RING, FULL, STAY, TWO>), dim3(blocks), dim3(64 * WI * WJ), lds, stream, g,
                 (int)tiles);
    return FRCNN_OK;
}

template <typename T, bool AKC, bool BKC, int BI, int BJ, int WI, int WJ, int RING>
static int dn_launch_ring(const DnGemm& g, unsigned blocks, hipStream_t stream) {
    const bool full = !g.partial && (g.e.bias || g.e.pre || g.e.residual || g.e.act != FRCNN_ACT_NONE || g.e.out_f32);
    if constexpr (AKC)          // d_weight's product has none of it
        if (full) return dn_launch_kernel<T, AKC, BKC, BI, BJ, WI, WJ, RING, true, false>(g, blocks, stream);
    if (g.low_a || g.low_b) return dn_launch_kernel<T, AKC, BKC, BI, BJ, WI, WJ, RING, false, true>(g, blocks, stream);
    return dn_launch_kernel<T, AKC, BKC, BI, BJ, WI, WJ, RING, false, false>(g, blocks, stream);
}

template <typename T, bool AKC, bool BKC, int BI, int BJ, int WI, int WJ>
static int dn_launch_tiles(const DnGemm& g, unsigned blocks, hipStream_t stream) {
    if constexpr (AKC && BKC && BI < 256)       // of 128 x 256 a compute unit holds one in any case
        if (BJ == 256 || blocks <= DN_CUS) return dn_launch_ring<T, AKC, BKC, BI, BJ, WI, WJ, 6>(g, blocks, stream);
    if constexpr (!(AKC && BKC && BJ == 256 && BI < 256)) return dn_launch_ring<T, AKC, BKC, BI, BJ, WI, WJ, 4>(g, blocks, stream);
    return FRCNN_E_UNSUPPORTED;
}

template <typename T, bool AKC, bool BKC>
static int dn_launch_gemm(const DnPlan& pl, const DnGemm& g, hipStream_t stream) {
    if (pl.bi == 0) {
        if (!dn_grid(pl.tiles_j, 64 * DN_FW)) return FRCNN_E_UNSUPPORTED;
        if constexpr (AKC) {
            const dim3 grid((unsigned)pl.tiles_j, (unsigned)pl.splits);
            const dim3 block(64 * DN_FW);
            if (g.low_a) {
                if (g.I <= 16) FRCNN_LAUNCH((dense_few_rows_kernel<T, BKC, 1, true>), grid, block, 0, stream, g);
                else FRCNN_LAUNCH((dense_few_rows_kernel<T, BKC, 2, true>), grid, block, 0, stream, g);
            } else {
                if (g.I <= 16) FRCNN_LAUNCH((dense_few_rows_kernel<T, BKC, 1, false>), grid, block, 0, stream, g);
                else FRCNN_LAUNCH((dense_few_rows_kernel<T, BKC, 2, false>), grid, block, 0, stream, g);
            }
        }
        return FRCNN_OK;
    }
    const long long blocks = pl.tiles_i * pl.tiles_j * pl.splits;
    if (!dn_grid(blocks, pl.bj == 256 ? 512 : 256)) return FRCNN_E_UNSUPPORTED;
    if (pl.bi == 256) return dn_launch_tiles<T, AKC, BKC, 256, 256, 2, 4>(g, (unsigned)blocks, stream);
    if (pl.bj == 256) return dn_launch_tiles<T, AKC, BKC, 128, 256, 2, 4>(g, (unsigned)blocks, stream);
    if (pl.bi == 128) return dn_launch_tiles<T, AKC, BKC, 128, 128, 2, 2>(g, (unsigned)blocks, stream);
    return dn_launch_tiles<T, AKC, BKC, 64, 128, 1, 4>(g, (unsigned)blocks, stream);
}

static size_t dn_up(size_t b) { return (b + 255) / 256 * 256; }

// A matrix in memory as rows of `cols` values.  padded: its rows are whole pieces with zeros behind `cols`.
// low: elements to the low part of a dz in two parts, scale and low_scale what undoes their factors
struct DnMatrix { const void* p; long long rows, cols, ld; bool padded; long long low = 0; float scale = 1.f, low_scale = 1.f; const float* scale_at = nullptr; };
static long long dn_pieces(long long n) { return (n + 7) / 8; }
// rows that start on 16 bytes, of whole 16-byte pieces
static bool dn_whole(const DnMatrix& m) {
    return reinterpret_cast<uintptr_t>(m.p) % 16 == 0 && m.ld % 8 == 0 && (m.padded || m.cols % 8 == 0) &&
           m.ld <= DN_MAX_LD;
}
static size_t dn_pack_bytes(long long rows, long long cols) {
    return dn_up((size_t)rows * (size_t)dn_pieces(cols) * 16);
}

// Copies of the matrices whose rows are not whole pieces, from `ws` on (which moves behind them): what has
// to be launched; a null matrix is left alone.
static int dn_pack(DnMatrix* a, DnMatrix* b, char*& ws, DnPacks& packs) {
    packs = DnPacks{};
    int n = 0;
    for (DnMatrix* m : {a, b}) {
        if (!m || dn_whole(*m)) continue;
        if (dn_pieces(m->cols) * 8 > DN_MAX_LD) return FRCNN_E_UNSUPPORTED;
        packs.of[n] = DnPack{m->p, ws, m->rows, m->cols, m->ld, dn_pieces(m->cols)};
        packs.blocks += (m->rows * packs.of[n].pieces + 255) / 256;
        if (n == 0) packs.blocks_first = packs.blocks;
        ws += dn_pack_bytes(m->rows, m->cols);
        *m = DnMatrix{packs.of[n].dst, m->rows, m->cols, packs.of[n].pieces * 8, true};
        ++n;
    }
    return dn_grid(packs.blocks, 256) ? FRCNN_OK : FRCNN_E_UNSUPPORTED;
}
template <typename T>
static int dn_launch_packs(const DnPacks& packs, hipStream_t stream) {
    if (packs.blocks) FRCNN_LAUNCH(dense_pack_kernel<T>, dim3((unsigned)packs.blocks), dim3(256), 0, stream, packs);
    return FRCNN_OK;
}

// D = A B^T: `a` holds A as [I][K] (akc) or [K][I], `b` B as [J][K] (bkc) or [K][J], packed where they have
// to be; the workspace holds the partial sums of a split reduction
static DnGemm dn_arguments(const DnPlan& pl, const DnMatrix& a, bool akc, const DnMatrix& b, bool bkc, const DnEpilogue& e,
                           void* ws) {
    DnGemm g{};
    g.I = akc ? a.rows : a.cols; g.J = bkc ? b.rows : b.cols; g.K = akc ? a.cols : a.rows;
    g.a = a.p; g.b = b.p; g.lda = a.ld; g.ldb = b.ld;
    g.outer_a = a.padded ? dn_pieces(g.I) * 8 : g.I;
    g.outer_b = b.padded ? dn_pieces(g.J) * 8 : g.J;
    g.k_slice = pl.k_slice; g.splits = pl.splits;
    g.tiles_i = (int)pl.tiles_i; g.tiles_j = (int)pl.tiles_j;
    g.partial = pl.splits > 1 ? (float*)ws : nullptr;
    g.low_a = a.low; g.low_b = b.low;
    const DnMatrix& dz = a.low ? a : b;
    g.scale = dz.scale; g.low_scale = dz.low_scale; g.scale_at = dz.scale_at;
    g.e = e;
    return g;
}
// joins what is split of one product or two
template <typename T>
static int dn_join(const DnGemm* a, const DnGemm* b, hipStream_t stream) {
    DnJoin j[2] = {};
    int n = 0;
    for (const DnGemm* g : {a, b})
        if (g && g->partial) j[n++] = DnJoin{g->partial, g->I, g->J, (g->I * ((g->J + 3) / 4) + 63) / 64, g->splits, g->e};
    if (n == 0) return FRCNN_OK;
    const long long blocks = j[0].blocks + j[1].blocks;
    if (!dn_grid(blocks, 64)) return FRCNN_E_UNSUPPORTED;
    FRCNN_LAUNCH(dense_join_kernel<T>, dim3((unsigned)blocks), dim3(64), 0, stream, j[0], j[1]);
    return FRCNN_OK;
}
template <typename T>
static int dn_product(const DnPlan& pl, const DnMatrix& a, bool akc, const DnMatrix& b, bool bkc, const DnEpilogue& e,
                      void* ws, hipStream_t stream) {
    if (pl.tiles_i > 0xFFFFFFF || pl.tiles_j > 0xFFFFFFF) return FRCNN_E_UNSUPPORTED;
    const DnGemm g = dn_arguments(pl, a, akc, b, bkc, e, ws);
    int rc;
    if (akc && bkc) rc = dn_launch_gemm<T, true, true>(pl, g, stream);
    else if (akc) rc = dn_launch_gemm<T, true, false>(pl, g, stream);
    else rc = dn_launch_gemm<T, false, false>(pl, g, stream);
    return rc != FRCNN_OK ? rc : dn_join<T>(&g, nullptr, stream);
}

// the plans of a backward's two products; whether they share a launch: both of small tiles, few enough workgroups to be
// on the chip at once (1,111 x 779 x 333 f16, dz in one part: 21.8 us for the call, 29.1 one after the other; 27.4 in two)
struct DnPair { DnPlan x, w; bool together; };
static DnPair dn_pair(int64_t M, int K, int N, bool kn, bool few) {
    DnPair p{dn_plan(M, K, N, true, kn, few), kn ? dn_plan(K, N, M, false, false, false) : dn_plan(N, K, M, false, false, false), false};
    auto small = [](const DnPlan& q) { return q.bi == 64 && q.tiles_i * q.tiles_j * q.splits <= 2 * DN_CUS; };
    p.together = small(p.x) && small(p.w);
    return p;
}
template <typename T, bool BKC, bool TWO>
static int dn_launch_pair(const DnGemm& x, const DnGemm& w, const DnBiasGrad& b, hipStream_t stream) {
    constexpr int lds = (BKC ? 6 : 4) * (64 + 128) * DN_SK * 2;
    static std::atomic<uint64_t> raised{0};
    if (!dn_raise_lds(reinterpret_cast<const void*>(dense_pair_kernel<T, BKC, TWO>), lds, raised)) return FRCNN_E_LAUNCH;
    const int tx = x.tiles_i * x.tiles_j * x.splits, tw = w.tiles_i * w.tiles_j * w.splits;
    const int tb = b.sums ? (b.N + 15) / 16 : 0;
    FRCNN_LAUNCH((dense_pair_kernel<T, BKC, TWO>), dim3((unsigned)(tx + tw + tb)), dim3(256), lds, stream, x, tx, w, tw, b);
    return dn_join<T>(&x, &w, stream);
}

// What a packed operand takes.  DN_ANY: rows anywhere; DN_ALIGNED: on 16 bytes
enum DnRows { DN_ANY, DN_ALIGNED };
static size_t dn_copy_bytes(long long rows, long long cols, DnRows r) {
    return r == DN_ALIGNED && cols % 8 == 0 ? 0 : dn_pack_bytes(rows, cols);
}
static size_t dn_copy_bytes(const DnMatrix& m) { return dn_whole(m) ? 0 : dn_pack_bytes(m.rows, m.cols); }

// the backward's workspace: both parts of dz, the largest |d_out| and the scale, the column sums, then what one product at
// a time needs
struct DnBwdPlan { bool copy; long long ldz; int cg; long long rows, blocks; size_t part_bytes, dz_bytes, sum_bytes; };
constexpr int DN_MOST = 256;                           // workgroups of dense_most_kernel

static DnBwdPlan dn_bwd_plan(long long M, int N, bool copy) {
    DnBwdPlan p{};
    if (M == 0) return p;                              // nothing to multiply: zeros are stored
    p.copy = copy;
    p.ldz = dn_pieces(N) * 8;
    if (M <= 256) {
        // one workgroup has all rows of 16 columns: no second launch for the sums (of 1,111 rows x 333
        // this took 26 us, the two launches 7.6 + 3.2)
        p.cg = 2;
        p.rows = M;
        p.blocks = 1;
    } else {
        // a workgroup takes 256 / cg rows at a time of 8 cg columns: two to eight such walks, as many
        // workgroups as fill the chip four times, at most 4,096 partial sums per column
        p.cg = 1;
        while (p.cg < 32 && p.cg < dn_pieces(N)) p.cg *= 2;
        const long long walk = 256 / p.cg, columns = (dn_pieces(N) + p.cg - 1) / p.cg;
        long long walks = M * columns / (walk * 4 * DN_CUS);
        walks = walks < 2 ? 2 : walks > 8 ? 8 : walks;
        while ((M + walk * walks - 1) / (walk * walks) > 4096) walks *= 2;
        p.rows = walk * walks;
        p.blocks = (M + p.rows - 1) / p.rows;
    }
    p.part_bytes = dn_up((size_t)M * (size_t)p.ldz * 2);
    p.dz_bytes = copy ? 2 * p.part_bytes + dn_up((DN_MOST + 1) * 4) : 0;
    p.sum_bytes = p.blocks > 1 ? dn_up((size_t)p.blocks * (size_t)N * 4) : 0;
    return p;
}

static bool dn_sizes(int64_t M, int K, int N) { return M >= 0 && K > 0 && N > 0; }
constexpr int64_t DN_MAX_ROWS = (1ll << 30) - 64;      // rows of 64 each: fewer than 2^24 workgroups of 256 threads
static bool dn_16bit(int dtype) { return dtype == FRCNN_DT_F16 || dtype == FRCNN_DT_BF16; }
static bool dn_even(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

template <typename T>
static int dn_zero(void* p, long long rows, long long cols, long long ld, hipStream_t s) {
    const long long groups = (rows * cols + 255) / 256;
    if (!dn_grid(groups, 256)) return FRCNN_E_UNSUPPORTED;
    FRCNN_LAUNCH(dense_zero_kernel<T>, dim3((unsigned)groups), dim3(256), 0, s, (T*)p, rows, cols, ld);
    return FRCNN_OK;
}

template <typename T>
static int dn_forward(DnMatrix x, DnMatrix w, bool bkc, bool few, const DnPlan& plan, const DnEpilogue& e, char* ws,
                      hipStream_t s) {
    if (!few) {
        DnPacks packs;
        int rc = dn_pack(&x, &w, ws, packs);
        if (rc == FRCNN_OK) rc = dn_launch_packs<T>(packs, s);
        if (rc != FRCNN_OK) return rc;
    }
    return dn_product<T>(plan, x, true, w, bkc, e, ws, s);
}

template <typename T>
static int dn_backward(const void* d_out, long long ldd, int d_dtype, const void* x, long long ldx, const void* w,
                       long long ldw, int w_layout, const void* pre, long long ldp, long long M, int K, int N,
                       int dtype, int act, void* d_x, long long lddx, void* d_w, long long lddw, void* d_bias,
                       char* ws, const DnBwdPlan& p, bool few, const DnPair& pair, hipStream_t s) {
    const bool kn = w_layout == FRCNN_W_KN;
    int rc = FRCNN_OK;
    if (M == 0) {
        if (d_w) rc = kn ? dn_zero<T>(d_w, K, N, lddw, s) : dn_zero<T>(d_w, N, K, lddw, s);
        if (rc == FRCNN_OK && d_bias) rc = dn_zero<T>(d_bias, 1, N, N, s);
        return rc;
    }
    if ((d_x || d_w) && dn_pieces(N) * 8 > DN_MAX_LD) return FRCNN_E_UNSUPPORTED;
    void* dz = p.copy && (d_x || d_w) ? ws : nullptr;
    char* rest = ws + p.dz_bytes + p.sum_bytes;
    // d_out's values or 0 are dz where d_out has the products' type and act is none or ReLU; else dz is in two parts,
    // in float16 with the low part up by 2^11 (its own 11 bits also below the normal range) and both down by two (act'
    // reaches 1.13: no overflow), or by what brings a float32 d_out into range
    const bool two = dz && (d_dtype != dtype || act > FRCNN_ACT_RELU), f16 = dtype == FRCNN_DT_F16;
    const float scale = f16 ? 0.5f : 1.0f, low_up = f16 ? 2048.0f : 1.0f;
    DnMatrix z = dz ? DnMatrix{dz, M, N, p.ldz, true} : DnMatrix{d_out, M, N, ldd, false};
    if (two) {
        z.low = (long long)(p.part_bytes / 2);
        z.scale = 1.0f / scale;
        z.low_scale = 1.0f / low_up;
    }
    DnMatrix mx{x, M, K, ldx, false}, mw = kn ? DnMatrix{w, K, N, ldw, false} : DnMatrix{w, N, K, ldw, false};
    DnPacks packs;
    rc = dn_pack(d_x && !few ? &mw : nullptr, d_w ? &mx : nullptr, rest, packs);
    if (rc != FRCNN_OK) return rc;
    float* most = two && f16 && d_dtype == FRCNN_DT_F32 ? reinterpret_cast<float*>(ws + 2 * p.part_bytes) : nullptr;
    int n_most = 0;
    if (most) {
        z.scale_at = most + DN_MOST;
        const long long blocks = (M * dn_pieces(N) + 255) / 256;
        n_most = blocks < DN_MOST ? (int)blocks : DN_MOST;
        FRCNN_LAUNCH(dense_most_kernel, dim3((unsigned)n_most), dim3(256), 0, s, (const float*)d_out, ldd, M, N, most);
    }
    DnBiasGrad bias{};
    if (d_bias || dz) {
        DnDz q{};
        q.d_out = d_out; q.ldd = ldd; q.pre = pre; q.ldp = ldp; q.dz = dz; q.ldz = p.ldz;
        q.M = M; q.N = N; q.act = act; q.cg = p.cg; q.rows = p.rows; q.row_blocks = p.blocks;
        q.low = z.low; q.scale = scale; q.low_up = low_up;
        q.most = most; q.n_most = n_most; q.back = most ? most + DN_MOST : nullptr;
        if (p.blocks == 1) q.d_bias = d_bias;
        else q.sums = d_bias ? reinterpret_cast<float*>(ws + p.dz_bytes) : nullptr;
        q.blocks = p.blocks * ((dn_pieces(N) + p.cg - 1) / p.cg);
        const long long blocks = q.blocks + packs.blocks;
        if (!dn_grid(blocks, 256)) return FRCNN_E_UNSUPPORTED;
        if (d_dtype == FRCNN_DT_F32)
            FRCNN_LAUNCH((dense_dz_kernel<T, float>), dim3((unsigned)blocks), dim3(256), 0, s, q, packs);
        else
            FRCNN_LAUNCH((dense_dz_kernel<T, T>), dim3((unsigned)blocks), dim3(256), 0, s, q, packs);
        if (q.sums) {
            bias = DnBiasGrad{q.sums, d_bias, (int)p.blocks, N};
            if (!pair.together)
                FRCNN_LAUNCH(dense_bias_grad_kernel<T>, dim3((unsigned)((N + 15) / 16)), dim3(1024), 0, s, bias);
        }
    } else {
        rc = dn_launch_packs<T>(packs, s);
        if (rc != FRCNN_OK) return rc;
    }
    DnEpilogue e{};
    if (pair.together) {
        e.out = d_x; e.ldo = lddx;
        const DnGemm gx = dn_arguments(pair.x, z, true, mw, kn, e, rest);
        e.out = d_w; e.ldo = lddw;
        char* behind = rest + dn_up(pair.x.partial_bytes);
        const DnGemm gw = kn ? dn_arguments(pair.w, mx, false, z, false, e, behind)
                             : dn_arguments(pair.w, z, false, mx, false, e, behind);
        if (two) return kn ? dn_launch_pair<T, true, true>(gx, gw, bias, s) : dn_launch_pair<T, false, true>(gx, gw, bias, s);
        return kn ? dn_launch_pair<T, true, false>(gx, gw, bias, s) : dn_launch_pair<T, false, false>(gx, gw, bias, s);
    }
    if (d_x) {
        e.out = d_x; e.ldo = lddx;
        rc = dn_product<T>(pair.x, z, true, mw, kn, e, rest, s);
        if (rc != FRCNN_OK) return rc;
    }
    if (d_w) {
        e.out = d_w; e.ldo = lddw;
        rc = kn ? dn_product<T>(pair.w, mx, false, z, false, e, rest, s) : dn_product<T>(pair.w, z, false, mx, false, e, rest, s);
    }
    return rc;
}

}  // namespace frcnn

using namespace frcnn;

// what a forward's packed operands and partial sums take
static size_t dn_fwd_bytes(const DnPlan& plan, bool few, size_t copies) { return dn_up(plan.partial_bytes) + (few ? 0 : copies); }
extern "C" size_t frcnn_dense_fwd_workspace_bytes(int64_t M, int K, int N, int w_layout, int aligned) {
    if (!dn_sizes(M, K, N) || M == 0 || M > DN_MAX_ROWS) return 0;
    const DnRows x = aligned & 1 ? DN_ALIGNED : DN_ANY, w = aligned & 2 ? DN_ALIGNED : DN_ANY;
    const bool kn = w_layout == FRCNN_W_KN;
    const size_t copy_x = dn_copy_bytes(M, K, x), copy_w = kn ? dn_copy_bytes(K, N, w) : dn_copy_bytes(N, K, w);
    const bool few = dn_few(M, N, K, !kn, copy_w == 0), few_whole = dn_few(M, N, K, !kn, true);
    size_t need = dn_fwd_bytes(dn_plan(M, N, K, true, !kn, few), few, copy_x + copy_w);
    if (few != few_whole) {                            // W may be whole after all
        const size_t other = dn_fwd_bytes(dn_plan(M, N, K, true, !kn, few_whole), few_whole, copy_x);
        if (need < other) need = other;
    }
    return need;
}

extern "C" int frcnn_dense_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, int w_layout, const void* bias,
                               const void* residual, int64_t ldr, int64_t M, int K, int N, int dtype, int act,
                               void* out, int64_t ldo, int out_dtype, void* pre, int64_t ldp, void* workspace,
                               size_t workspace_bytes, frcnn_stream_t stream) {
    if (!dn_sizes(M, K, N) || !dn_16bit(dtype) || (out_dtype != dtype && out_dtype != FRCNN_DT_F32))
        return FRCNN_E_BADARG;
    if (act < FRCNN_ACT_NONE || act > FRCNN_ACT_SILU || (w_layout != FRCNN_W_KN && w_layout != FRCNN_W_NK))
        return FRCNN_E_BADARG;
    if (M > DN_MAX_ROWS) return FRCNN_E_UNSUPPORTED;
    if (M == 0) return FRCNN_OK;
    const bool kn = w_layout == FRCNN_W_KN;
    if (!x || !w || !out || ldx < K || ldw < (kn ? N : K) || ldo < N) return FRCNN_E_BADARG;
    if ((residual && ldr < N) || (pre && ldp < N)) return FRCNN_E_BADARG;
    if (!dn_even(x, 2) || !dn_even(w, 2) || !dn_even(bias, 2) || !dn_even(residual, 2) || !dn_even(pre, 2) ||
        !dn_even(out, out_dtype == FRCNN_DT_F32 ? 4 : 2))
        return FRCNN_E_BADARG;
    const DnMatrix mx{x, M, K, ldx, false}, mw = kn ? DnMatrix{w, K, N, ldw, false} : DnMatrix{w, N, K, ldw, false};
    const bool few = dn_few(M, N, K, !kn, dn_whole(mw));
    const DnPlan plan = dn_plan(M, N, K, true, !kn, few);
    const size_t need = dn_fwd_bytes(plan, few, dn_copy_bytes(mx) + dn_copy_bytes(mw));
    if (need && (!workspace || workspace_bytes < need || !dn_even(workspace, 16))) return FRCNN_E_WORKSPACE;
    DnEpilogue e{};
    e.bias = bias; e.residual = residual; e.pre = pre; e.out = out;
    e.ldr = ldr; e.ldp = ldp; e.ldo = ldo; e.act = act; e.out_f32 = out_dtype == FRCNN_DT_F32;
    return dtype == FRCNN_DT_BF16
               ? dn_forward<__bf16>(mx, mw, !kn, few, plan, e, (char*)workspace, (hipStream_t)stream)
               : dn_forward<_Float16>(mx, mw, !kn, few, plan, e, (char*)workspace, (hipStream_t)stream);
}

// what a backward's dz, column sums, packed operands and partial sums (one product's at a time, or both) take
static size_t dn_bwd_bytes(const DnBwdPlan& p, const DnPair& pair, size_t copies) {
    const size_t x = dn_up(pair.x.partial_bytes), w = dn_up(pair.w.partial_bytes);
    return p.dz_bytes + p.sum_bytes + copies + (pair.together ? x + w : x > w ? x : w);
}
extern "C" size_t frcnn_dense_bwd_workspace_bytes(int64_t M, int K, int N, int w_layout, int aligned) {
    if (!dn_sizes(M, K, N) || M == 0 || M > DN_MAX_ROWS) return 0;
    const DnBwdPlan p = dn_bwd_plan(M, N, !(aligned & 4) || N % 8 != 0);
    const bool kn = w_layout == FRCNN_W_KN;
    const DnRows x = aligned & 1 ? DN_ALIGNED : DN_ANY, w = aligned & 2 ? DN_ALIGNED : DN_ANY;
    const size_t copy_x = dn_copy_bytes(M, K, x), copy_w = kn ? dn_copy_bytes(K, N, w) : dn_copy_bytes(N, K, w);
    const bool few = dn_few(M, K, N, kn, copy_w == 0), few_whole = dn_few(M, K, N, kn, true);
    size_t need = dn_bwd_bytes(p, dn_pair(M, K, N, kn, few), copy_x + (few ? 0 : copy_w));
    if (few != few_whole) {                            // W may be whole after all
        const size_t other = dn_bwd_bytes(p, dn_pair(M, K, N, kn, few_whole), copy_x);
        if (need < other) need = other;
    }
    return need;
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
    if (M > DN_MAX_ROWS) return FRCNN_E_UNSUPPORTED;
    if (d_w && lddw < (kn ? N : K)) return FRCNN_E_BADARG;
    if (!dn_even(d_out, d_dtype == FRCNN_DT_F32 ? 4 : 2) || !dn_even(x, 2) || !dn_even(w, 2) || !dn_even(pre, 2) ||
        !dn_even(d_x, 2) || !dn_even(d_w, 2) || !dn_even(d_bias, 2))
        return FRCNN_E_BADARG;
    // dz is d_out itself where that is whole pieces in the products' type and no activation changes it
    const bool copy = act != FRCNN_ACT_NONE || d_dtype != dtype || !dn_whole(DnMatrix{d_out, M, N, ldd, false});
    if (M > 0) {
        if (!d_out || ldd < N) return FRCNN_E_BADARG;
        if (act != FRCNN_ACT_NONE && (!pre || ldp < N)) return FRCNN_E_BADARG;
        if (d_x && (!w || ldw < (kn ? N : K) || lddx < K)) return FRCNN_E_BADARG;
        if (d_w && (!x || ldx < K)) return FRCNN_E_BADARG;
    }
    const DnBwdPlan p = dn_bwd_plan(M, N, copy);
    bool few = false;
    DnPair pair{};
    if (M > 0) {
        const DnMatrix mx{x, M, K, ldx, false}, mw = kn ? DnMatrix{w, K, N, ldw, false} : DnMatrix{w, N, K, ldw, false};
        few = dn_few(M, K, N, kn, dn_whole(mw));
        pair = dn_pair(M, K, N, kn, few);
        pair.together = pair.together && d_x && d_w;
        if (!d_x) pair.x.partial_bytes = 0;
        if (!d_w) pair.w.partial_bytes = 0;
        const size_t need = dn_bwd_bytes(p, pair, (d_w ? dn_copy_bytes(mx) : 0) + (d_x && !few ? dn_copy_bytes(mw) : 0));
        if (need && (!workspace || workspace_bytes < need || !dn_even(workspace, 16))) return FRCNN_E_WORKSPACE;
    }
    return dtype == FRCNN_DT_BF16
               ? dn_backward<__bf16>(d_out, ldd, d_dtype, x, ldx, w, ldw, w_layout, pre, ldp, M, K, N, dtype, act,
                                     d_x, lddx, d_w, lddw, d_bias, (char*)workspace, p, few, pair, (hipStream_t)stream)
               : dn_backward<_Float16>(d_out, ldd, d_dtype, x, ldx, w, ldw, w_layout, pre, ldp, M, K, N, dtype, act,
                                       d_x, lddx, d_w, lddw, d_bias, (char*)workspace, p, few, pair, (hipStream_t)stream);
}
