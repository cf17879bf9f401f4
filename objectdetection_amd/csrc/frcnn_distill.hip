// Distillation of the class logits from a teacher's stored top logits, forward and backward.
//
// Row r with teacher logits t_j at labels i_j (j < k; an entry whose label is outside [0, V) or whose
// logit is -inf is not there) and student logits z_v (v < V), temperature T:
//     p = softmax(t / T) over the entries that are there,   q = softmax(z / T) over all V,
//     loss = w T^2 sum_j p_j (log p_j - log q_(i_j)),   d loss / d z_v = w T (q_v - sum_j p_j [i_j = v]).
// A row with w = 0 or no entry takes no part: its loss, lse and gradient are 0 whatever its logits are
// (with w = 0 they are not read).
//
// All sums are float32, relative to the row's maximum; log q is kept as (z - max) / T - log(sum), so the
// two large terms of z - lse never cancel: the backward takes maximum and sum from the logits again instead of the
// forward's lse, whose rounding would be in every q (2^-24 of lse: 2e-4 at logits of 1e4).  The gradient is written
// as c q first and the few listed labels are written again with their p subtracted; a label listed twice gets both.
//
// Memory is the bound: a logit is read once and its gradient written once.  A row stays in registers, as it
// lies in memory, between the three walks over it (maximum, sum, gradient): in those of a wave or a part of one
// (up to 512 pieces of 16 bytes, 64 entries), of a workgroup (up to 16,384 pieces).  Longer rows, and few long
// rows, are split: one launch leaves a maximum and a sum per chunk, a second one joins them in every workgroup
// and writes the chunk's gradient; in a backward without a workspace every workgroup walks its row itself.
#include "frcnn_common.h"

namespace frcnn {

constexpr int DS_MAX_K = 1024, DS_SHORT_K = 64;
constexpr float DS_LOG2E = 1.4426950408889634f;

struct DsArgs {
    const void* z; long long ldz;        // [rows,V]
    const void* t; int t_f32;            // [rows,k], float32 or the logits' type
    const int64_t* idx;                  // [rows,k]
    const float* weight;                 // [rows] or null
    const float* d_loss;                 // [rows] or null: the backward's upstream gradient
    float scale;                         // factor of the gradient when d_loss is null
    float temperature;
    long long rows; int V, k;
    float* loss; float* lse; void* grad; long long ldg;      // loss and lse: null in the backward
    float2* part; int chunks, nv;        // maximum and sum of each chunk of a split row; its vectors per thread
};

typedef unsigned int ds_u32x4 __attribute__((ext_vector_type(4)));

// sixteen bytes of a row, as they lie in memory: 4 float32 or 8 16-bit values
template <typename T>
struct DsVec {
    static constexpr int W = 16 / sizeof(T);
    ds_u32x4 b;
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (W == 4) {
            return __uint_as_float(b[i]);
        } else {
            const unsigned short h = (unsigned short)(b[i / 2] >> (16 * (i & 1)));
            return (float)__builtin_bit_cast(T, h);
        }
    }
    // keeps the compiler from holding the converted values from one walk over the row to the next
    __device__ __forceinline__ void renew() { asm volatile("" : "+v"(b)); }
    __device__ __forceinline__ void load(const T* p, int valid) {          // -inf behind the row's end
        if (valid >= W) {
            __builtin_memcpy(&b, p, 16);
        } else {
            T v[W];
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = i < valid ? p[i] : (T)-__builtin_inff();
            __builtin_memcpy(&b, v, 16);
        }
    }
    __device__ __forceinline__ void set(const float* f) {
        T v[W];
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = (T)f[i];
        __builtin_memcpy(&b, v, 16);
    }
    __device__ __forceinline__ void store(T* p, int valid) const {
        if (valid >= W) {
            __builtin_memcpy(p, &b, 16);
        } else {
            T v[W];
            __builtin_memcpy(v, &b, 16);
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (i < valid) p[i] = v[i];
        }
    }
};

// Over G neighbouring lanes, the same bits in each: within sixteen lanes the operand comes straight from a
// neighbour's register (quads, then halves and rows mirrored: what is met there is the same in a quad, in
// eight lanes), beyond by exchanging rows of sixteen and halves; with an LDS exchange per step
// short rows wait for LDS (500,000 rows of 64 bf16 classes and entries: 826 us; 257 this way).
template <int CTRL>
__device__ __forceinline__ float ds_dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <bool MAX>
__device__ __forceinline__ float ds_join(float a, float b) { return MAX ? fmaxf(a, b) : a + b; }
template <int G, bool MAX>
__device__ __forceinline__ float ds_lanes(float v) {
    static_assert(G >= 8 && G <= 64);
    v = ds_join<MAX>(v, ds_dpp<0xB1>(v));              // lanes 1 0 3 2
    v = ds_join<MAX>(v, ds_dpp<0x4E>(v));              // lanes 2 3 0 1
    v = ds_join<MAX>(v, ds_dpp<0x141>(v));             // eight mirrored
    if constexpr (G >= 16) v = ds_join<MAX>(v, ds_dpp<0x140>(v));      // sixteen mirrored
    if constexpr (G >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = ds_join<MAX>(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    if constexpr (G >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = ds_join<MAX>(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    return v;
}
__device__ __forceinline__ float ds_wave_max(float v) { return ds_lanes<64, true>(v); }
__device__ __forceinline__ float ds_wave_sum(float v) { return ds_lanes<64, false>(v); }
// over the workgroup, the same order for every thread; `sh` of BLOCK / 64 floats is used once per call
template <int BLOCK, bool MAX>
__device__ __forceinline__ float ds_block(float v, float* sh) {
    v = MAX ? ds_wave_max(v) : ds_wave_sum(v);
    if constexpr (BLOCK == 64) {
        return v;
    } else {
        if (lane_id() == 0) sh[wave_id()] = v;
        __syncthreads();
        v = sh[0];
#pragma unroll
        for (int w = 1; w < BLOCK / 64; ++w) v = MAX ? fmaxf(v, sh[w]) : v + sh[w];
        return v;
    }
}

// ---- the teacher's side of a row -----------------------------------------------------------------------
// LDS: per entry its label (-1: not there), its logit, then that relative to the largest one and over T, the student's logit there,
// and what its label gets: the sum of its entries' p, or a negative number where another entry of the label has
// it; with more than 64 entries also a table of twice as many places or more, in which entries of a label meet
constexpr int ds_slots(int k) {
    int n = 0;
    if (k > 64)
        for (n = 256; n < 2 * k; n *= 2) {}
    return n;
}
struct DsTeacher {
    int* label; float* t; float* z; float* p; int* key; int* first;
    __device__ __forceinline__ DsTeacher(void* lds, int k)
        : label((int*)lds), t((float*)lds + k), z((float*)lds + 2 * k), p((float*)lds + 3 * k), key((int*)lds + 4 * k),
          first(key + ds_slots(k)) {}
};
static size_t ds_lds_bytes(int k) { return (size_t)k * 16 + (size_t)ds_slots(k) * 8; }

template <typename T>
__device__ __forceinline__ float ds_teacher_logit(const DsArgs& a, long long at) {
    return a.t_f32 ? ((const float*)a.t)[at] : (float)((const T*)a.t)[at];
}

// label, logit (as stored: dividing by T first would round what the maximum cancels, or overflow) and the student's
// logit of the row's entries, by the whole workgroup; whether this wave met one
template <typename T, int BLOCK>
__device__ __forceinline__ bool ds_teacher_load(const DsArgs& a, long long row, DsTeacher e) {
    const T* z = (const T*)a.z + row * a.ldz;
    bool any = false;
    for (int j = threadIdx.x; j < a.k; j += BLOCK) {
        const int64_t i = a.idx[row * a.k + j];
        const float t = ds_teacher_logit<T>(a, row * a.k + j);
        const bool there = i >= 0 && i < a.V && !(t == -__builtin_inff());
        e.label[j] = there ? (int)i : -1;
        e.t[j] = t;
        if (there) {
            any = true;
            e.z[j] = (float)z[i];
        }
    }
    return __ballot(any) != 0;
}
// makes t relative to the largest one, over T, and returns the log of the sum of e^t, by one wave
__device__ __forceinline__ float ds_teacher_sum(DsTeacher e, int k, float inv_t) {
    const int lane = lane_id();
    float top = -__builtin_inff(), s = 0.f;
    for (int j = lane; j < k; j += 64) top = fmaxf(top, e.label[j] >= 0 ? e.t[j] : -__builtin_inff());
    top = ds_wave_max(top);
    for (int j = lane; j < k; j += 64) {
        const float t = (e.t[j] - top) * inv_t;
        e.t[j] = t;
        if (e.label[j] >= 0) s += __builtin_amdgcn_exp2f(t * DS_LOG2E);
    }
    return logf(ds_wave_sum(s));
}
// over the workgroup, behind a barrier after sh[wave] was set
template <int BLOCK>
__device__ __forceinline__ bool ds_any(const int* sh) {
    int any = sh[0];
#pragma unroll
    for (int w = 1; w < BLOCK / 64; ++w) any |= sh[w];
    return any != 0;
}

// sum_j p_j (log p_j - log q_j) with log q = (z - z_max) / T - log_s, by the same wave
__device__ __forceinline__ float ds_row_loss(const DsArgs& a, DsTeacher e, float log_sum, float inv_t, float z_max,
                                             float log_s) {
    float l = 0.f;
    for (int j = lane_id(); j < a.k; j += 64) {
        if (e.label[j] < 0) continue;
        const float log_p = e.t[j] - log_sum, p = __builtin_amdgcn_exp2f(log_p * DS_LOG2E);
        const float log_q = (e.z[j] - z_max) * inv_t - log_s;
        if (!(p == 0.f)) l += p * (log_p - log_q);
    }
    return ds_wave_sum(l);
}

// e.p for the labels in [v0, v1), by the whole workgroup.  Up to 64 entries: one wave compares each with all
// of them one by one (from a register of another lane: an LDS read per comparison costs the whole row its
// latency), and entries of the same label come to the same sum.  More: that would be the square of their number, so
// each looks for its label's place in the table, and the first entry of a label adds up the later ones, in their
// order (4,096 rows x 65,536, 1,024 entries: 313 us; 1,917 by comparing all with all).
template <int BLOCK>
__device__ __forceinline__ void ds_listed_sums(DsTeacher e, int k, const float* sh_log_sum, long long v0, long long v1) {
    if (k <= 64) {
        if (wave_id() != 0) return;
        const float log_sum = *sh_log_sum;             // this wave's own
        const int lane = lane_id();
        const int mine = lane < k ? e.label[lane] : -1;
        const float p = lane < k ? __builtin_amdgcn_exp2f((e.t[lane] - log_sum) * DS_LOG2E) : 0.f;
        float sum = 0.f;
        for (int n = 0; n < k; ++n) {
            const int other = __builtin_amdgcn_readlane(mine, n);
            const float q = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), n));
            sum += other == mine ? q : 0.f;
        }
        if (lane < k) e.p[lane] = mine >= 0 ? sum : -1.0f;
        return;
    }
    const int tid = threadIdx.x, slots = ds_slots(k), shift = __builtin_clz(slots) + 1;
    for (int n = tid; n < slots; n += BLOCK) {
        e.key[n] = -1;
        e.first[n] = k;
    }
    __syncthreads();
    const float log_sum = *sh_log_sum;
    for (int j = tid; j < k; j += BLOCK) {             // places; e.p: the entry's place
        const int label = e.label[j];
        if (label < v0 || label >= v1) {
            e.p[j] = -1.0f;
            continue;
        }
        int n = (int)(((unsigned)label * 2654435761u) >> shift);
        while (true) {                                 // ends: there are more places than labels
            const int held = atomicCAS(&e.key[n], -1, label);
            if (held == -1 || held == label) break;
            n = (n + 1) & (slots - 1);
        }
        atomicMin(&e.first[n], j);
        e.p[j] = __int_as_float(n);
    }
    __syncthreads();
    for (int j = tid; j < k; j += BLOCK) {             // the later ones form a chain: key -2 - j, e.p -2 - j of the next
        if (e.p[j] < 0.f) continue;
        const int n = __float_as_int(e.p[j]);
        if (e.first[n] == j) continue;
        const int held = atomicExch(&e.key[n], -2 - j);
        e.p[j] = held >= 0 ? -1.0f : (float)held;
    }
    __syncthreads();
    for (int j = tid; j < k; j += BLOCK) {
        if (e.p[j] < 0.f) continue;
        const int head = e.key[__float_as_int(e.p[j])], label = e.label[j];
        float sum = __builtin_amdgcn_exp2f((e.t[j] - log_sum) * DS_LOG2E);
        int length = 0;
        for (int n = head; n < -1 && length <= 16; ++length) n = (int)e.p[-2 - n];
        if (length <= 16) {                            // the chain's order is chance: the smallest number first
            for (int from = j, m = 0; m < length; ++m) {
                int next = k;
                for (int n = head; n < -1; n = (int)e.p[-2 - n])
                    if (-2 - n > from && -2 - n < next) next = -2 - n;
                sum += __builtin_amdgcn_exp2f((e.t[next] - log_sum) * DS_LOG2E);
                from = next;
            }
        } else {
            for (int n = j + 1; n < k; ++n)
                if (e.label[n] == label) sum += __builtin_amdgcn_exp2f((e.t[n] - log_sum) * DS_LOG2E);
        }
        e.p[j] = sum;
    }
}

// writes the gradient at the listed labels in [v0, v1)
template <typename T, typename Q>
__device__ __forceinline__ void ds_listed(DsTeacher e, int k, float c, T* grad, long long v0, long long v1, int tid,
                                          int block, Q q_of) {
    for (int j = tid; j < k; j += block) {
        const int i = e.label[j];
        const float p = e.p[j];
        if (i >= v0 && i < v1 && !(p < 0.f)) grad[i] = (T)(c * (q_of(e.z[j]) - p));      // also a NaN
    }
}

template <typename T>
__device__ __forceinline__ void ds_zero(T* grad, long long v0, long long v1, int tid, int block) {
    DsVec<T> o;
    o.b = ds_u32x4{0, 0, 0, 0};
    for (long long v = v0 + tid * DsVec<T>::W; v < v1; v += block * DsVec<T>::W)
        o.store(grad + v, v1 - v > DsVec<T>::W ? DsVec<T>::W : (int)(v1 - v));
}

// ---- rows of a few classes: a class and an entry per lane, G lanes per row -----------------------------
// Up to 16 classes and entries, or rows of less than 16 bytes (1,000,000 rows of 8 f32 classes with 4 entries
// 33.8 us, 3.3 TB/s).
template <typename T, bool FORWARD, int G>
__global__ void __launch_bounds__(256) distill_small_kernel(DsArgs a) {
    __shared__ __attribute__((aligned(16))) float2 entry[256];        // label and p of a row's entries
    const int l = threadIdx.x & (G - 1), first = lane_id() & ~(G - 1);
    const long long row = (long long)blockIdx.x * (256 / G) + threadIdx.x / G;
    if (row >= a.rows) return;                         // whole groups of lanes leave
    const float inv_t = 1.0f / a.temperature, ninf = -__builtin_inff(), f = inv_t * DS_LOG2E;
    const float w = a.weight ? a.weight[row] : 1.0f;
    const bool mine = l < a.V;
    const float z = mine && w != 0.f ? (float)((const T*)a.z)[row * a.ldz + l] : ninf;
    int label = -1;
    float t = ninf;
    if (l < a.k) {
        const int64_t i = a.idx[row * a.k + l];
        t = ds_teacher_logit<T>(a, row * a.k + l);
        if (i >= 0 && i < a.V && !(t == ninf)) label = (int)i;
    }
    const float top = ds_lanes<G, true>(label >= 0 ? t : ninf), m = ds_lanes<G, true>(z);
    const bool any = (__ballot(label >= 0) >> first & (~0ull >> (64 - G))) != 0;
    const float te = label >= 0 ? __builtin_amdgcn_exp2f((t - top) * f) : 0.f;
    const float ts = ds_lanes<G, false>(te);
    const float s = ds_lanes<G, false>(mine ? __builtin_amdgcn_exp2f((z - m) * f) : 0.f);
    const bool part = w != 0.f && any;
    const float log_sum = logf(ts), log_s = logf(s);
    const float log_p = (t - top) * inv_t - log_sum, p = label >= 0 ? __builtin_amdgcn_exp2f(log_p * DS_LOG2E) : 0.f;
    const float zi = __shfl(z, first + (label >= 0 ? label : 0));
    if (FORWARD) {
        const float loss =
            ds_lanes<G, false>(label >= 0 && !(p == 0.f) ? p * (log_p - ((zi - m) * inv_t - log_s)) : 0.f);
        if (l == 0) {
            a.loss[row] = part ? w * (a.temperature * a.temperature) * loss : 0.f;
            a.lse[row] = part ? m * inv_t + log_s : 0.f;
        }
        if (!a.grad) return;
    }
    entry[threadIdx.x] = make_float2(__int_as_float(label), p);       // read by the same wave
    __builtin_amdgcn_wave_barrier();
    float listed = 0.f;                                // the p of the entries that name this lane's class
    for (int j = 0; j < a.k; j += 2) {
        const float4 two = *reinterpret_cast<const float4*>(&entry[threadIdx.x - l + j]);
        if (__float_as_int(two.x) == l) listed += two.y;
        if (__float_as_int(two.z) == l) listed += two.w;
    }
    const float c = w * a.temperature * (a.d_loss ? a.d_loss[row] : a.scale);
    const float log_q = (z - m) * inv_t - log_s;
    if (mine)
        ((T*)a.grad)[row * a.ldg + l] = (T)(part ? c * (__builtin_amdgcn_exp2f(log_q * DS_LOG2E) - listed) : 0.f);
}

// ---- short rows with up to 64 entries: G lanes per row, NV pieces of 16 bytes per lane -------------------
// What such a row costs is latency and issued instructions (1,000,000 x 21: vector instructions issue in 0.8 of the
// cycles, memory at 3.0 TB/s): several rows per wave, its entries and weight loaded before anything is decided, no
// barrier.  1,000,000 x 21 f32 with 8 entries 83 us (156 with a lane per class),
// 300,000 x 91 bf16 50 us (203 with a workgroup per row), 100,000 x 1,203 f32 with 32 entries 190 us, 5.3 TB/s
// (351).  The piece that would end behind the row is the row's last 16 bytes instead: what it
// shares with its neighbour is left out of the sums and stored twice with the same value.
template <typename T, bool FORWARD, int G, int NV>
__global__ void __launch_bounds__(256) distill_short_kernel(DsArgs a) {
    constexpr int W = DsVec<T>::W, E = DS_SHORT_K / G;            // entries per lane
    __shared__ __attribute__((aligned(16))) float2 entry[256 / G][DS_SHORT_K + 2];       // label and p
    const int l = threadIdx.x & (G - 1), first = lane_id() & ~(G - 1), rl = threadIdx.x / G;
    const long long row = (long long)blockIdx.x * (256 / G) + rl;
    if (row >= a.rows) return;                         // whole groups of lanes leave
    const float inv_t = 1.0f / a.temperature, ninf = -__builtin_inff(), f = inv_t * DS_LOG2E;
    const float w = a.weight ? a.weight[row] : 1.0f;
    const float up = a.d_loss ? a.d_loss[row] : a.scale;
    const T* z = (const T*)a.z + row * a.ldz;
    int label[E];
    float t[E], zi[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        label[e] = -1;
        t[e] = ninf;
        zi[e] = 0.f;
        if (G * e >= a.k) continue;
        const int j = l + G * e, at = j < a.k ? j : a.k - 1;
        const int64_t i = a.idx[row * a.k + at];
        t[e] = ds_teacher_logit<T>(a, row * a.k + at);
        if (j < a.k && i >= 0 && i < a.V && !(t[e] == ninf)) label[e] = (int)i;
    }
    DsVec<T> x[NV];
    int from[NV], dup[NV];                             // the piece's place; how many of its values belong to others
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = (l + G * i) * W;
        from[i] = v + W <= a.V ? v : a.V - W;
        dup[i] = v >= a.V ? W : v - from[i];
        x[i].b = ds_u32x4{0, 0, 0, 0};
        if (w != 0.f) x[i].load(z + from[i], W);
    }
    if (w != 0.f) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (label[e] >= 0) zi[e] = (float)z[label[e]];
    }
    float top = ninf, m = ninf;
    bool any = false;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        any |= label[e] >= 0;
        top = fmaxf(top, label[e] >= 0 ? t[e] : ninf);
    }
    top = ds_lanes<G, true>(top);
    any = (__ballot(any) >> first & (~0ull >> (64 - G))) != 0;
    auto value = [&](int i, int n) { return n < dup[i] ? ninf : x[i][n]; };
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int n = 0; n < W; ++n) m = fmaxf(m, value(i, n));
    m = ds_lanes<G, true>(m);
    float ts = 0.f, s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) ts += label[e] >= 0 ? __builtin_amdgcn_exp2f((t[e] - top) * f) : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int n = 0; n < W; ++n) s += __builtin_amdgcn_exp2f((value(i, n) - m) * f);
    const float log_sum = logf(ds_lanes<G, false>(ts));
    s = ds_lanes<G, false>(s);
    const float log_s = logf(s);
    const bool part = w != 0.f && any;
    float p[E];
    float loss = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float log_p = (t[e] - top) * inv_t - log_sum;
        p[e] = label[e] >= 0 ? __builtin_amdgcn_exp2f(log_p * DS_LOG2E) : 0.f;
        if (label[e] >= 0 && !(p[e] == 0.f)) loss += p[e] * (log_p - ((zi[e] - m) * inv_t - log_s));
    }
    if (FORWARD) {
        loss = ds_lanes<G, false>(loss);
        if (l == 0) {
            a.loss[row] = part ? w * (a.temperature * a.temperature) * loss : 0.f;
            a.lse[row] = part ? m * inv_t + log_s : 0.f;
        }
        if (!a.grad) return;
    }
    T* grad = (T*)a.grad + row * a.ldg;
    const float c = w * a.temperature * up, cq = c / s;
    auto relative = [&](float v) { return __builtin_amdgcn_exp2f((v - m) * f); };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float q[W];
#pragma unroll
        for (int n = 0; n < W; ++n) q[n] = part ? cq * relative(x[i][n]) : 0.f;
        x[i].set(q);
        if (dup[i] < W) x[i].store(grad + from[i], W);
    }
    if (!part) return;                                 // whole groups of lanes
    // entries of the same label add up the same values in the same order and store the same result, behind
    // what the same wave stored above
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (G * e < a.k) entry[rl][l + G * e] = make_float2(__int_as_float(label[e]), p[e]);
        sum[e] = 0.f;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
    for (int j = 0; j < a.k; j += 2) {
        const float4 two = *reinterpret_cast<const float4*>(&entry[rl][j]);
        const int i0 = __float_as_int(two.x), i1 = __float_as_int(two.z);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (G * e >= a.k) continue;
            sum[e] += i0 == label[e] ? two.y : 0.f;
            sum[e] += i1 == label[e] ? two.w : 0.f;
        }
    }
    const float scale = 1.0f / s;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (label[e] >= 0) grad[label[e]] = (T)(c * (relative(zi[e]) * scale - sum[e]));
}

// ---- a whole row in the registers of one workgroup: up to BLOCK * NV vectors ------------------------------
// 4,096 rows x 65,536 bf16 with 64 entries 213 us, 5.05 TB/s: what a copy reaches
template <typename T, int BLOCK, int NV>
__global__ void __launch_bounds__(BLOCK) distill_row_kernel(DsArgs a) {
    extern __shared__ __attribute__((aligned(16))) char ds_lds[];
    __shared__ float sh_m[BLOCK / 64], sh_s[BLOCK / 64], sh_t;
    __shared__ int sh_any[BLOCK / 64];
    constexpr int W = DsVec<T>::W;
    const int tid = threadIdx.x;
    const long long row = blockIdx.x;
    const T* z = (const T*)a.z + row * a.ldz;
    T* grad = a.grad ? (T*)a.grad + row * a.ldg : nullptr;
    const float w = a.weight ? a.weight[row] : 1.0f, inv_t = 1.0f / a.temperature;
    if (w == 0.f) {
        if (tid == 0 && a.loss) { a.loss[row] = 0.f; a.lse[row] = 0.f; }
        if (grad) ds_zero(grad, 0, a.V, tid, BLOCK);
        return;
    }
    DsVec<T> x[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = (tid + BLOCK * i) * W;
        x[i].load(z + v, a.V - v);
    }
    const DsTeacher e(ds_lds, a.k);
    const bool some = ds_teacher_load<T, BLOCK>(a, row, e);        // while the row arrives
    if (lane_id() == 0) sh_any[wave_id()] = some;
    float m = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) m = fmaxf(m, x[i][j]);
    m = ds_block<BLOCK, true>(m, sh_m);
    if constexpr (BLOCK == 64) __syncthreads();
    if (!ds_any<BLOCK>(sh_any)) {
        if (tid == 0 && a.loss) { a.loss[row] = 0.f; a.lse[row] = 0.f; }
        if (grad) ds_zero(grad, 0, a.V, tid, BLOCK);
        return;
    }
    float log_sum = 0.f;
    if (wave_id() == 0) {
        log_sum = ds_teacher_sum(e, a.k, inv_t);
        if (tid == 0) sh_t = log_sum;
    }
    const float f = inv_t * DS_LOG2E;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float part = 0.f;
        x[i].renew();
#pragma unroll
        for (int j = 0; j < W; ++j) part += __builtin_amdgcn_exp2f((x[i][j] - m) * f);
        s += part;
    }
    if (grad) ds_listed_sums<BLOCK>(e, a.k, &sh_t, 0, a.V);
    s = ds_block<BLOCK, false>(s, sh_s);
    const float log_s = logf(s);
    if (wave_id() == 0 && a.loss) {
        const float l = ds_row_loss(a, e, log_sum, inv_t, m, log_s);
        if (tid == 0) {
            a.loss[row] = w * (a.temperature * a.temperature) * l;
            a.lse[row] = m * inv_t + log_s;
        }
    }
    if (!grad) return;
    const float c = w * a.temperature * (a.d_loss ? a.d_loss[row] : a.scale), cq = c / s;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        int t = tid;
        // a large workgroup has 128 registers per lane: the places are not kept in them from the loads on
        // (2,048 rows x 131,072 bf16: 253 us; 280 with 68 bytes per lane waiting in memory)
        if constexpr (BLOCK == 1024) asm volatile("" : "+v"(t));
        const int v = (t + BLOCK * i) * W;
        float q[W];
        x[i].renew();
#pragma unroll
        for (int j = 0; j < W; ++j) q[j] = cq * __builtin_amdgcn_exp2f((x[i][j] - m) * f);
        x[i].set(q);
        x[i].store(grad + v, a.V - v);
    }
    __syncthreads();                                   // the stores of c q come before those of the listed labels
    ds_listed(e, a.k, c, grad, 0, a.V, tid, BLOCK,
              [&](float zi) { return __builtin_amdgcn_exp2f((zi - m) * f) / s; });
}

// ---- a chunk of a row per workgroup --------------------------------------------------------------------
// of 4 vectors per thread, of one where the rows are few and their chunks would not fill the chip (one row of
// 131,072 f32: 8.7 us for the two launches, latency of loads and sums)
constexpr int DS_CHUNK_BLOCK = 256;
template <typename T, int BLOCK, int NV> constexpr int ds_chunk() { return BLOCK * NV * DsVec<T>::W; }

template <typename T, int NV>
__global__ void __launch_bounds__(DS_CHUNK_BLOCK) distill_part_kernel(DsArgs a) {
    __shared__ float sh_m[DS_CHUNK_BLOCK / 64], sh_s[DS_CHUNK_BLOCK / 64];
    constexpr int W = DsVec<T>::W;
    const int tid = threadIdx.x, chunk = blockIdx.x;
    const long long row = blockIdx.y;
    if (a.weight && a.weight[row] == 0.f) return;
    const T* z = (const T*)a.z + row * a.ldz;
    const long long v0 = (long long)chunk * ds_chunk<T, DS_CHUNK_BLOCK, NV>();
    DsVec<T> x[NV];
    float m = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const long long v = v0 + (tid + DS_CHUNK_BLOCK * i) * W, left = a.V - v;
        x[i].load(z + v, left > W ? W : (int)left);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) m = fmaxf(m, x[i][j]);
    m = ds_block<DS_CHUNK_BLOCK, true>(m, sh_m);
    const float f = DS_LOG2E / a.temperature;
    const float base = m == -__builtin_inff() ? 0.f : m;    // a chunk of -inf alone has the sum 0
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) s += __builtin_amdgcn_exp2f((x[i][j] - base) * f);
    s = ds_block<DS_CHUNK_BLOCK, false>(s, sh_s);
    if (tid == 0) a.part[row * a.chunks + chunk] = float2{m, s};
}

// joins the row's partial sums; in the forward chunk 0 writes loss and lse
template <typename T, int BLOCK, int NV>
__global__ void __launch_bounds__(BLOCK) distill_chunk_kernel(DsArgs a) {
    extern __shared__ __attribute__((aligned(16))) char ds_lds[];
    __shared__ float sh_t, sh_m, sh_s;
    __shared__ int sh_any[BLOCK / 64];
    constexpr int W = DsVec<T>::W;
    const int tid = threadIdx.x, chunk = blockIdx.x;
    const long long row = blockIdx.y;
    const T* z = (const T*)a.z + row * a.ldz;
    T* grad = a.grad ? (T*)a.grad + row * a.ldg : nullptr;
    const long long v0 = (long long)chunk * ds_chunk<T, BLOCK, NV>(), v1 = v0 + ds_chunk<T, BLOCK, NV>() < a.V ? v0 + ds_chunk<T, BLOCK, NV>() : a.V;
    const float w = a.weight ? a.weight[row] : 1.0f, inv_t = 1.0f / a.temperature;
    if (w == 0.f) {
        if (chunk == 0 && tid == 0 && a.loss) { a.loss[row] = 0.f; a.lse[row] = 0.f; }
        if (grad) ds_zero(grad, v0, v1, tid, BLOCK);
        return;
    }
    DsVec<T> x[NV];
    if (grad) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const long long v = v0 + (tid + BLOCK * i) * W, left = a.V - v;
            x[i].load(z + v, left > W ? W : (int)left);
        }
    }
    const DsTeacher e(ds_lds, a.k);
    const bool some = ds_teacher_load<T, BLOCK>(a, row, e);
    if (lane_id() == 0) sh_any[wave_id()] = some;
    if (wave_id() == 1) {                              // every workgroup joins the chunks in the same order
        float m = -__builtin_inff(), s = 0.f;
        for (int c = lane_id(); c < a.chunks; c += 64) m = fmaxf(m, a.part[row * a.chunks + c].x);
        m = ds_wave_max(m);
        for (int c = lane_id(); c < a.chunks; c += 64) {
            const float2 q = a.part[row * a.chunks + c];
            const float d = q.x == m ? 0.f : q.x - m;  // also where both are infinite
            s += q.y * __builtin_amdgcn_exp2f(d * (inv_t * DS_LOG2E));
        }
        s = ds_wave_sum(s);
        if (lane_id() == 0) { sh_m = m; sh_s = m == -__builtin_inff() ? __builtin_nanf("") : s; }
    }
    __syncthreads();
    if (!ds_any<BLOCK>(sh_any)) {
        if (chunk == 0 && tid == 0 && a.loss) { a.loss[row] = 0.f; a.lse[row] = 0.f; }
        if (grad) ds_zero(grad, v0, v1, tid, BLOCK);
        return;
    }
    float log_sum = 0.f;
    if (wave_id() == 0) {
        log_sum = ds_teacher_sum(e, a.k, inv_t);
        if (tid == 0) sh_t = log_sum;
    }
    const float m = sh_m, s = sh_s;
    if (chunk == 0 && wave_id() == 0 && a.loss) {
        const float log_s = logf(s), l = ds_row_loss(a, e, log_sum, inv_t, m, log_s);
        if (tid == 0) {
            a.loss[row] = w * (a.temperature * a.temperature) * l;
            a.lse[row] = m * inv_t + log_s;
        }
    }
    if (!grad) return;
    ds_listed_sums<BLOCK>(e, a.k, &sh_t, v0, v1);
    const float c = w * a.temperature * (a.d_loss ? a.d_loss[row] : a.scale), cq = c / s;
    const float f = inv_t * DS_LOG2E;
    auto relative = [&](float zi) { return __builtin_amdgcn_exp2f((zi - m) * f); };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const long long v = v0 + (tid + BLOCK * i) * W, left = a.V - v;
        float q[W];
#pragma unroll
        for (int j = 0; j < W; ++j) q[j] = cq * relative(x[i][j]);
        x[i].set(q);
        x[i].store(grad + v, left > W ? W : (int)left);
    }
    __syncthreads();
    ds_listed(e, a.k, c, grad, v0, v1, tid, BLOCK, [&](float zi) { return relative(zi) / s; });
}

// ---- the same backward without a workspace ---------------------------------------------------------------
// There is nowhere to leave sums: every workgroup walks the whole row for them, 4 vectors per thread at a time with a
// running maximum and the sum relative to it, and writes the gradient of its chunk, reading that again.  Bound by the
// walk's latency where rows are few (one of 131,072 f32 15.6 us, 9 in two launches with a workspace; 64 of 131,072 bf16
// 30 and 16), by memory else (2,048 of 131,072 f32 624 and 565).
constexpr int DS_WALK_BLOCK = 512, DS_WALK_VECTORS = 4;

template <typename T>
__global__ void __launch_bounds__(DS_WALK_BLOCK) distill_walk_kernel(DsArgs a) {
    extern __shared__ __attribute__((aligned(16))) char ds_lds[];
    __shared__ float sh_t, sh_m[DS_WALK_BLOCK / 64], sh_s[DS_WALK_BLOCK / 64];
    __shared__ int sh_any[DS_WALK_BLOCK / 64];
    constexpr int W = DsVec<T>::W, BLOCK = DS_WALK_BLOCK, NV = DS_WALK_VECTORS;
    const int tid = threadIdx.x;
    const long long row = blockIdx.y, per = (long long)a.nv * (BLOCK * NV * W), v0 = blockIdx.x * per;
    const long long v1 = v0 + per < a.V ? v0 + per : a.V;
    const T* z = (const T*)a.z + row * a.ldz;
    T* grad = (T*)a.grad + row * a.ldg;
    const float w = a.weight ? a.weight[row] : 1.0f, inv_t = 1.0f / a.temperature, f = inv_t * DS_LOG2E;
    if (w == 0.f) return ds_zero(grad, v0, v1, tid, BLOCK);
    const DsTeacher e(ds_lds, a.k);
    const bool some = ds_teacher_load<T, BLOCK>(a, row, e);
    if (lane_id() == 0) sh_any[wave_id()] = some;
    __syncthreads();
    if (!ds_any<BLOCK>(sh_any)) return ds_zero(grad, v0, v1, tid, BLOCK);
    if (wave_id() == 0) {
        const float log_sum = ds_teacher_sum(e, a.k, inv_t);
        if (tid == 0) sh_t = log_sum;
    }
    DsVec<T> x[NV];
    auto load = [&](long long at, long long end) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const long long v = at + (tid + BLOCK * i) * W, left = end - v;
            x[i].load(z + v, left > W ? W : (int)left);
        }
    };
    // A maximum of -inf is taken as 0: nothing but -inf was met, and its sum is 0.
    float m = -__builtin_inff(), s = 0.f;
    for (long long at = 0; at < a.V; at += BLOCK * NV * W) {
        load(at, a.V);
        float top = m, part = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) top = fmaxf(top, x[i][j]);
        const float base = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) part += __builtin_amdgcn_exp2f((x[i][j] - base) * f);
        s = s * __builtin_amdgcn_exp2f((m - base) * f) + part;
        m = top;
    }
    const float most = ds_block<BLOCK, true>(m, sh_m);
    s = ds_block<BLOCK, false>(s * __builtin_amdgcn_exp2f(m == most ? 0.f : (m - most) * f), sh_s);
    if (most == -__builtin_inff()) s = __builtin_nanf("");
    ds_listed_sums<BLOCK>(e, a.k, &sh_t, v0, v1);
    const float c = w * a.temperature * a.d_loss[row], cq = c / s;
    auto relative = [&](float zi) { return __builtin_amdgcn_exp2f((zi - most) * f); };
    for (long long at = v0; at < v1; at += BLOCK * NV * W) {
        load(at, v1);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const long long v = at + (tid + BLOCK * i) * W, left = v1 - v;
            float q[W];
#pragma unroll
            for (int j = 0; j < W; ++j) q[j] = cq * relative(x[i][j]);
            x[i].set(q);
            x[i].store(grad + v, left > W ? W : (int)left);
        }
    }
    __syncthreads();                                   // the stores of c q come before those of the listed labels
    ds_listed(e, a.k, c, grad, v0, v1, tid, BLOCK, [&](float zi) { return relative(zi) / s; });
}

// ---- host --------------------------------------------------------------------------------------------
// rows that one workgroup can hold, and long rows of which there are too few to fill the chip
static long long ds_vectors(int V, int dtype) { return (V + (dtype == FRCNN_DT_F32 ? 4 : 8) - 1) / (dtype == FRCNN_DT_F32 ? 4 : 8); }
// vectors per thread of a chunk
static int ds_chunk_vectors(long long rows, int V, int dtype) {
    const long long four = (ds_vectors(V, dtype) + DS_CHUNK_BLOCK * 4 - 1) / (DS_CHUNK_BLOCK * 4);
    return rows * four <= 256 ? 1 : 4;
}
static long long ds_chunks(long long rows, int V, int dtype) {
    const long long c = (long long)DS_CHUNK_BLOCK * ds_chunk_vectors(rows, V, dtype);
    return (ds_vectors(V, dtype) + c - 1) / c;
}
static bool ds_split(long long rows, int V, int dtype) {
    const long long n = ds_vectors(V, dtype);
    return n > 16384 || (n >= 4 * 1024 && rows * ((n + 1023) / 1024) <= 1024);
}
static int ds_group(int V, int k) {
    int g = 1;
    while (g < V || g < k) g *= 2;
    return g;
}
// rows of which a wave takes one or more
static bool ds_short(int V, int k, int dtype) { return k <= DS_SHORT_K && ds_vectors(V, dtype) <= 512; }

// rows r .. r + n - 1 of a call
template <typename T>
static DsArgs ds_rows(const DsArgs& a, long long r, long long n) {
    DsArgs b = a;
    b.rows = n;
    b.z = (const T*)a.z + r * a.ldz;
    b.t = (const char*)a.t + r * a.k * (a.t_f32 ? 4 : (long long)sizeof(T));
    b.idx = a.idx + r * a.k;
    if (a.weight) b.weight = a.weight + r;
    if (a.d_loss) b.d_loss = a.d_loss + r;
    if (a.loss) { b.loss = a.loss + r; b.lse = a.lse + r; }
    if (a.grad) b.grad = (T*)a.grad + r * a.ldg;
    if (a.part) b.part = a.part + r * a.chunks;
    return b;
}

template <typename T, bool FORWARD, int G>
static int ds_launch_small(const DsArgs& a, hipStream_t s) {
    FRCNN_LAUNCH((distill_small_kernel<T, FORWARD, G>), dim3((unsigned)((a.rows + 256 / G - 1) / (256 / G))), dim3(256),
                 0, s, a);
    return FRCNN_OK;
}
template <typename T, bool FORWARD, int G, int NV>
static int ds_launch_short(const DsArgs& a, hipStream_t s) {
    FRCNN_LAUNCH((distill_short_kernel<T, FORWARD, G, NV>), dim3((unsigned)((a.rows + 256 / G - 1) / (256 / G))),
                 dim3(256), 0, s, a);
    return FRCNN_OK;
}
template <typename T, int BLOCK, int NV>
static int ds_launch_row(const DsArgs& a, hipStream_t s) {
    FRCNN_LAUNCH((distill_row_kernel<T, BLOCK, NV>), dim3((unsigned)a.rows), dim3(BLOCK), ds_lds_bytes(a.k),
                 s, a);
    return FRCNN_OK;
}
template <typename T, int BLOCK, int NV>
static int ds_launch_chunk(const DsArgs& a, hipStream_t s) {
    FRCNN_LAUNCH((distill_part_kernel<T, NV>), dim3((unsigned)a.chunks, (unsigned)a.rows), dim3(BLOCK), 0, s, a);
    const dim3 grid(a.grad ? (unsigned)a.chunks : 1u, (unsigned)a.rows);           // without a gradient: the loss alone
    FRCNN_LAUNCH((distill_chunk_kernel<T, BLOCK, NV>), grid, dim3(BLOCK), ds_lds_bytes(a.k), s, a);
    return FRCNN_OK;
}
template <typename T>
static int ds_launch_walk(const DsArgs& a, hipStream_t s) {
    FRCNN_LAUNCH(distill_walk_kernel<T>, dim3((unsigned)a.chunks, (unsigned)a.rows), dim3(DS_WALK_BLOCK), ds_lds_bytes(a.k),
                 s, a);
    return FRCNN_OK;
}

template <typename T, bool FORWARD>
static int ds_run(const DsArgs& a, int dtype, hipStream_t s) {
    const long long n = ds_vectors(a.V, dtype);
    if (ds_short(a.V, a.k, dtype)) {
        // a value per lane up to 16 classes (300,000 x 12 f32 with 4 entries 23.7 us, 28.1 in pieces; 40 classes
        // with 20 entries 112 us, 56 in pieces), and where a row is less than a piece
        const int g = ds_group(a.V, a.k);
        if (g <= 8) return ds_launch_small<T, FORWARD, 8>(a, s);
        if (g <= 16) return ds_launch_small<T, FORWARD, 16>(a, s);
        if (a.V < DsVec<T>::W)
            return g <= 32 ? ds_launch_small<T, FORWARD, 32>(a, s) : ds_launch_small<T, FORWARD, 64>(a, s);
        if (n <= 8) return ds_launch_short<T, FORWARD, 8, 1>(a, s);
        if (n <= 16) return ds_launch_short<T, FORWARD, 16, 1>(a, s);
        if (n <= 64) return ds_launch_short<T, FORWARD, 16, 4>(a, s);
        if (n <= 128) return ds_launch_short<T, FORWARD, 32, 4>(a, s);
        if (n <= 256) return ds_launch_short<T, FORWARD, 64, 4>(a, s);
        return ds_launch_short<T, FORWARD, 64, 8>(a, s);
    }
    // a short row with more entries is one wave's up to 192 of them (16,384 x 1,000: with 100 entries 35 us, 50 by
    // four waves; with 1,000 entries 755 and 307)
    const bool one_wave = a.k <= 192;
    if (a.chunks) {
        if (!a.part) return ds_launch_walk<T>(a, s);
        return a.nv == 1 ? ds_launch_chunk<T, DS_CHUNK_BLOCK, 1>(a, s) : ds_launch_chunk<T, DS_CHUNK_BLOCK, 4>(a, s);
    }
    if (n <= 64 && one_wave) return ds_launch_row<T, 64, 1>(a, s);
    if (n <= 256 && one_wave) return ds_launch_row<T, 64, 4>(a, s);
    if (n <= 256) return ds_launch_row<T, 256, 1>(a, s);
    if (n <= 1024) return ds_launch_row<T, 256, 4>(a, s);
    if (n <= 2048) return ds_launch_row<T, 256, 8>(a, s);
    if (n <= 4096) return ds_launch_row<T, 512, 8>(a, s);
    if (n <= 8192) return ds_launch_row<T, 512, 16>(a, s);
    return ds_launch_row<T, 1024, 16>(a, s);
}

// a launch at a time: rows are the grid's second dimension where rows have chunks (65,535 at most), else
// workgroups of up to 1,024 threads (fewer than 2^32 threads in a launch)
template <bool FORWARD>
static int ds_dispatch(DsArgs a, int dtype, hipStream_t s) {
    const bool chunked = !ds_short(a.V, a.k, dtype) && ds_split(a.rows, a.V, dtype);
    if (!chunked) a.part = nullptr;
    if (chunked && a.part) {
        a.nv = ds_chunk_vectors(a.rows, a.V, dtype);
        a.chunks = (int)ds_chunks(a.rows, a.V, dtype);
    } else if (chunked) {                              // nv: steps of the walk per chunk; up to 512 workgroups for few rows
        const long long step = DS_WALK_BLOCK * DS_WALK_VECTORS, steps = (ds_vectors(a.V, dtype) + step - 1) / step;
        const long long most = a.rows < 512 ? 512 / a.rows : 1;
        a.nv = (int)((steps + most - 1) / most);
        a.chunks = (int)((steps + a.nv - 1) / a.nv);
    }
    const long long at_once = chunked ? 65535 : 1 << 21;
    for (long long r = 0; r < a.rows; r += at_once) {
        const long long n = a.rows - r < at_once ? a.rows - r : at_once;
        const int rc = dtype == FRCNN_DT_F32   ? ds_run<float, FORWARD>(ds_rows<float>(a, r, n), dtype, s)
                       : dtype == FRCNN_DT_F16 ? ds_run<_Float16, FORWARD>(ds_rows<_Float16>(a, r, n), dtype, s)
                                               : ds_run<__bf16, FORWARD>(ds_rows<__bf16>(a, r, n), dtype, s);
        if (rc != FRCNN_OK) return rc;
    }
    return FRCNN_OK;
}

static int ds_check(const void* z, int64_t ldz, int dtype, const void* t, int t_dtype, const int64_t* idx,
                    int64_t rows, int V, int k, float temperature) {
    if (rows < 0 || V <= 0 || k <= 0 || ldz < V) return FRCNN_E_BADARG;
    if (dtype != FRCNN_DT_F32 && dtype != FRCNN_DT_F16 && dtype != FRCNN_DT_BF16) return FRCNN_E_BADARG;
    if (t_dtype != dtype && t_dtype != FRCNN_DT_F32) return FRCNN_E_BADARG;
    if (!(temperature >= 1e-18f && temperature <= 1e18f)) return FRCNN_E_BADARG;   // its square is a float32 too
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

extern "C" size_t frcnn_distill_workspace_bytes(int64_t rows, int V, int k, int dtype) {
    if (rows <= 0 || V <= 0 || k <= 0 || !ds_split(rows, V, dtype)) return 0;
    return (size_t)rows * (size_t)ds_chunks(rows, V, dtype) * sizeof(float2);
}

extern "C" int frcnn_distill_loss(const void* logits, int64_t ldz, int dtype, const void* top_values, int t_dtype,
                                  const int64_t* top_index, const float* weight, int64_t rows, int V, int k,
                                  float temperature, float grad_scale, float* loss, float* lse, void* d_logits,
                                  int64_t ldg, void* workspace, size_t workspace_bytes, frcnn_stream_t stream) {
    const int rc = ds_check(logits, ldz, dtype, top_values, t_dtype, top_index, rows, V, k, temperature);
    if (rc != FRCNN_OK || rows == 0) return rc;
    if (!loss || !lse || (d_logits && ldg < V)) return FRCNN_E_BADARG;
    const size_t need = frcnn_distill_workspace_bytes(rows, V, k, dtype);
    if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 8))
        return FRCNN_E_WORKSPACE;
    DsArgs a{};
    a.z = logits; a.ldz = ldz; a.t = top_values; a.idx = top_index; a.weight = weight; a.scale = grad_scale;
    a.temperature = temperature; a.rows = rows; a.V = V; a.k = k;
    a.loss = loss; a.lse = lse; a.grad = d_logits; a.ldg = ldg; a.t_f32 = t_dtype == FRCNN_DT_F32;
    a.part = (float2*)workspace;
    return ds_dispatch<true>(a, dtype, (hipStream_t)stream);
}

extern "C" int frcnn_distill_bwd_ws(const float* d_loss, const void* logits, int64_t ldz, int dtype,
                                    const void* top_values, int t_dtype, const int64_t* top_index, const float* lse,
                                    const float* weight, int64_t rows, int V, int k, float temperature,
                                    void* d_logits, int64_t ldg, void* workspace, size_t workspace_bytes,
                                    frcnn_stream_t stream) {
    const int rc = ds_check(logits, ldz, dtype, top_values, t_dtype, top_index, rows, V, k, temperature);
    if (rc != FRCNN_OK || rows == 0) return rc;
    if (!d_loss || !lse || !d_logits || ldg < V) return FRCNN_E_BADARG;
    const size_t need = frcnn_distill_workspace_bytes(rows, V, k, dtype);
    if (workspace && need && (workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 8))
        return FRCNN_E_WORKSPACE;
    DsArgs a{};
    a.z = logits; a.ldz = ldz; a.t = top_values; a.idx = top_index; a.weight = weight; a.d_loss = d_loss;
    a.temperature = temperature; a.rows = rows; a.V = V; a.k = k;
    a.grad = d_logits; a.ldg = ldg; a.t_f32 = t_dtype == FRCNN_DT_F32;
    a.part = (float2*)workspace;
    return ds_dispatch<false>(a, dtype, (hipStream_t)stream);
}

extern "C" int frcnn_distill_bwd(const float* d_loss, const void* logits, int64_t ldz, int dtype,
                                 const void* top_values, int t_dtype, const int64_t* top_index, const float* lse,
                                 const float* weight, int64_t rows, int V, int k, float temperature, void* d_logits,
                                 int64_t ldg, frcnn_stream_t stream) {
    return frcnn_distill_bwd_ws(d_loss, logits, ldz, dtype, top_values, t_dtype, top_index, lse, weight, rows, V, k,
                                temperature, d_logits, ldg, nullptr, 0, stream);
}
