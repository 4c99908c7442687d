// The two ends of a residual block (qcnn_op_norm_res; kernels_norm_*.hip make a type of it each): post norm, gate, scaled
// residual addition and the next block's norm in one pass over the row.
//
//   s = sum_j y[index[r][j]];  h = beta x + alpha act(gate) post(s);  n = pre(h)
//
// A row is owned by LPR threads and stays in their registers as float32 from the first load to the last store: every
// input is read once and every output written once, the floor of the operator.  A thread holds CPT chunks of 16 bytes,
// chunk c of a row belonging to thread c mod LPR, so that neighbouring threads touch neighbouring addresses.
// Loads and stores take any alignment; only the chunk that the end of a row cuts goes by elements.
// The memory bounds it.  Measured here and below: a call of a captured graph of calls, median of 9, inputs cold: 16384 x 4096 bfloat16 with
// a gate, 5 arrays: 136 to 139 us, 4.8 to 4.9 TB/s; 4096 x 2048 half, eight gathered rows each: 43 to 47 us, 4.0 to 4.3 TB/s; one row of
// 4096: 3.7 us, the latency of one load, two sums and one store.
// Statistics are float32 (the variance as the mean of the squared distances from the mean, from the registers).
#pragma once
#include "block_ops.h"

namespace qcnn {

// 16 bytes of a row as they stand in memory.
template <typename T>
struct Chunk {
    static constexpr int VE = 16 / sizeof(T);
    u32x4 raw;
    // elements [0, left) of the chunk exist; the others read as zero
    __device__ __forceinline__ void load(const T *p, int left)
    {
        raw = u32x4{0, 0, 0, 0};
        if (left >= VE) {
            raw = *(const u32x4_any *)p;
        } else {
            T t[VE];
            __builtin_memset(t, 0, 16);
#pragma unroll
            for (int i = 0; i < VE - 1; ++i)
                if (i < left) t[i] = p[i];
            __builtin_memcpy(&raw, t, 16);
        }
    }
    template <bool STREAM>
    __device__ __forceinline__ void store(T *p, int left) const
    {
        if (left >= VE) {
            if constexpr (STREAM)
                __builtin_nontemporal_store(raw, (u32x4_any *)p);
            else
                *(u32x4_any *)p = raw;
        } else {
            T t[VE];
            __builtin_memcpy(t, &raw, 16);
#pragma unroll
            for (int i = 0; i < VE - 1; ++i)
                if (i < left) p[i] = t[i];
        }
    }
    __device__ __forceinline__ void get(float (&v)[VE]) const
    {
        T t[VE];
        __builtin_memcpy(t, &raw, 16);
#pragma unroll
        for (int i = 0; i < VE; ++i) v[i] = to_f32(t[i]);
    }
    __device__ __forceinline__ void set(const float (&v)[VE])
    {
        T t[VE];
#pragma unroll
        for (int i = 0; i < VE; ++i) from_f32(v[i], t[i]);
        __builtin_memcpy(&raw, t, 16);
    }
};

// Sum over the LPR threads of a row; `red` holds one float for each wave, two sets used in turn so that one barrier
// a sum is enough.
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float *red, int &turn)
{
#pragma unroll
    for (int o = (LPR < 64 ? LPR : 64) / 2; o; o >>= 1) v += __shfl_xor(v, o);
    if constexpr (LPR > 64) {
        constexpr int NW = LPR / 64;
        float *set = red + turn * NW;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) set[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) v += set[i];
    }
    return v;
}

// VE weights of a norm from element `at` on, of T or float32; a missing vector is `none` everywhere.
template <typename T, int VE = Chunk<T>::VE>
__device__ __forceinline__ void norm_weights(const void *p, int w_type, int at, int left, float none, float add, float (&o)[VE])
{
    if (!p) {
#pragma unroll
        for (int i = 0; i < VE; ++i) o[i] = none;
        return;
    }
    if (w_type == QCNN_F32) {
        constexpr int N = VE / 4;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            Chunk<float> c;
            float f[4];
            c.load((const float *)p + at + 4 * j, left - 4 * j);
            c.get(f);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[4 * j + i] = f[i];
        }
    } else {
        Chunk<T> c;
        c.load((const T *)p + at, left);
        c.get(o);
    }
#pragma unroll
    for (int i = 0; i < VE; ++i) o[i] += add;
}

// tanh from e^2u; near zero, where 1 - 2 / (1 + e^2u) cancels, its Taylor polynomial to u^9 (the next term is
// 2^-24 of the value at 0.3).
__device__ __forceinline__ float tanh_of(float u)
{
    const float q = u * u;
    const float p = fmaf(q, fmaf(q, fmaf(q, fmaf(q, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
    const float e = 1.f - 2.f / (1.f + __expf(2.f * u));
    return fabsf(u) < 0.3f ? u * p : e;
}

template <typename T, int LPR, int CPT, bool STREAM>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void k_norm_res(const qcnn_norm_res_t a)
{
    typedef Chunk<T> C;
    constexpr int VE = C::VE, BLOCK = LPR > 256 ? LPR : 256, RPB = BLOCK / LPR;
    __shared__ float red[LPR > 64 ? 2 * (LPR / 64) : 1];
    int turn = 0;
    const int t = threadIdx.x % LPR;
    const size_t r = (size_t)blockIdx.x * RPB + threadIdx.x / LPR;
    if (RPB > 1 && r >= (size_t)a.rows) return;  // whole rows leave (LPR <= 64: no barrier follows)
    const int d = a.d;
    const float inv_d = 1.f / (float)d;
    float v[CPT][VE];

    // (What v holds behind the row's end is not zero once a norm has subtracted a mean there: the sums leave it out.)
    const auto norm = [&](int kind, const void *w, const void *b, float eps) {
        if (kind == QCNN_NORM_NONE) return;
        float mean = 0.f;
        if (kind == QCNN_NORM_LAYER) {
            float s = 0.f;
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
                const int left = d - (c * LPR + t) * VE;
#pragma unroll
                for (int i = 0; i < VE; ++i) s += i < left ? v[c][i] : 0.f;
            }
            mean = row_sum<LPR>(s, red, turn) * inv_d;
        }
        float q = 0.f;
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
            const int left = d - (c * LPR + t) * VE;
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                const float u = i < left ? v[c][i] - mean : 0.f;
                q = fmaf(u, u, q);
            }
        }
        const float inv = 1.f / sqrtf(row_sum<LPR>(q, red, turn) * inv_d + eps);
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
            const int at = (c * LPR + t) * VE, left = d - at;
            if (left <= 0) continue;
            float wv[VE], bv[VE];
            norm_weights<T>(w, a.w_type, at, left, 1.f, a.w_offset, wv);
            norm_weights<T>(b, a.w_type, at, left, 0.f, 0.f, bv);
#pragma unroll
            for (int i = 0; i < VE; ++i) v[c][i] = fmaf((v[c][i] - mean) * inv, wv[i], bv[i]);
        }
    };

    // the row's other inputs are asked for before the first sum waits, where registers for them are left
    constexpr bool EARLY = CPT * LPR <= 2048;
    C xr[EARLY ? CPT : 1], gr[EARLY ? CPT : 1];
    const T *x = (const T *)a.x + r * a.ldx;
    const T *g = a.gate ? (const T *)a.gate + ((unsigned)r / (unsigned)a.gate_rows) * a.ldg : nullptr;
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
        const int at = (c * LPR + t) * VE;
        if (EARLY && at < d) xr[EARLY ? c : 0].load(x + at, d - at);
        if (EARLY && at < d && g) gr[EARLY ? c : 0].load(g + at, d - at);
#pragma unroll
        for (int i = 0; i < VE; ++i) v[c][i] = 0.f;
    }
    if (a.y) {
        if (!a.index) {
            const T *y = (const T *)a.y + r * a.ldy;
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
                const int at = (c * LPR + t) * VE;
                if (at >= d) continue;
                C p;
                p.load(y + at, d - at);
                p.get(v[c]);
            }
        } else {
            const int32_t *ix = a.index + r * a.parts;
#pragma unroll 2
            for (int j = 0; j < a.parts; ++j) {
                const int k = ix[j];
                const bool have = k >= 0 && k < a.y_rows;
                const T *y = (const T *)a.y + (size_t)(have ? k : 0) * a.ldy;  // an index outside reads row 0 and drops it
#pragma unroll
                for (int c = 0; c < CPT; ++c) {
                    const int at = (c * LPR + t) * VE;
                    if (at >= d) continue;
                    C p;
                    p.load(y + at, d - at);
                    float u[VE];
                    p.get(u);
#pragma unroll
                    for (int i = 0; i < VE; ++i) v[c][i] += have ? u[i] : 0.f;
                }
            }
        }
        norm(a.post, a.post_w, a.post_b, a.post_eps);
    }
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
        const int at = (c * LPR + t) * VE;
        if (at >= d) continue;
        float u[VE];
        if (g) {
            if (!EARLY) gr[0].load(g + at, d - at);
            gr[EARLY ? c : 0].get(u);
            if (a.act == QCNN_GATE_TANH) {
#pragma unroll
                for (int i = 0; i < VE; ++i) u[i] = tanh_of(u[i]);
            } else if (a.act != QCNN_GATE_LINEAR) {
#pragma unroll
                for (int i = 0; i < VE; ++i) u[i] = (a.act == QCNN_GATE_SILU ? u[i] : 1.f) * sigmoid(u[i]);
            }
#pragma unroll
            for (int i = 0; i < VE; ++i) v[c][i] *= u[i];
        }
        if (!EARLY) xr[0].load(x + at, d - at);
        xr[EARLY ? c : 0].get(u);
#pragma unroll
        for (int i = 0; i < VE; ++i) v[c][i] = a.y ? fmaf(a.beta, u[i], a.alpha * v[c][i]) : a.beta * u[i];
        if (a.h) {
            C o;
            o.set(v[c]);
            o.template store<STREAM>((T *)a.h + r * a.ldh + at, d - at);
        }
    }
    if (!a.n) return;
    norm(a.pre, a.pre_w, a.pre_b, a.pre_eps);
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
        const int at = (c * LPR + t) * VE;
        if (at >= d) continue;
        C o;
        o.set(v[c]);
        o.template store<STREAM>((T *)a.n + r * a.ldn + at, d - at);
    }
}

template <typename T, int LPR, int CPT>
static hipError_t run(const qcnn_norm_res_t &a, hipStream_t s)
{
    constexpr int BLOCK = LPR > 256 ? LPR : 256, RPB = BLOCK / LPR;
    // Outputs from 8 MB on are written past the caches: 2048 x 8192 bf16 42.8 -> 38.1 us, 16384 x 4096 112.5 -> 109.6
    // (with a gate 142 -> 138), 4096 x 2048 half of eight parts 47.0 -> 43.4.  With copies of h and n right behind, 16384 x 4096 210 -> 206,
    // but 4096 x 1024 (16 MB) 19.2 -> 19.6; 256 x 4096 10.5 either way.
    const bool stream = (size_t)a.rows * a.d * sizeof(T) * ((a.h != nullptr) + (a.n != nullptr)) >= (size_t)8 << 20;
    // A launch's threads have to stay below 2^32: more rows take several, that part where a row of gate does, or inside one.
    const long long most = (0xffffffffu / BLOCK) * (long long)RPB, gate_rows = a.gate ? a.gate_rows : 1;
    qcnn_norm_res_t part = a;
    for (long long done = 0; done < a.rows; done += part.rows) {
        const long long fit = gate_rows <= most ? most / gate_rows * gate_rows : gate_rows - done % gate_rows < most ? gate_rows - done % gate_rows : most;
        part.rows = (int)(a.rows - done < fit ? a.rows - done : fit);
        part.x = (const T *)a.x + (size_t)done * a.ldx;
        if (a.index)
            part.index = a.index + (size_t)done * a.parts;
        else if (a.y)
            part.y = (const T *)a.y + (size_t)done * a.ldy;
        if (a.gate) part.gate = (const T *)a.gate + (size_t)(done / gate_rows) * a.ldg;
        if (a.h) part.h = (T *)a.h + (size_t)done * a.ldh;
        if (a.n) part.n = (T *)a.n + (size_t)done * a.ldn;
        const unsigned blocks = ((unsigned)part.rows + RPB - 1) / RPB;
        if (stream)
            k_norm_res<T, LPR, CPT, true><<<blocks, BLOCK, 0, s>>>(part);
        else
            k_norm_res<T, LPR, CPT, false><<<blocks, BLOCK, 0, s>>>(part);
        const hipError_t launched = hipGetLastError();
        if (launched != hipSuccess) return launched;
    }
    return hipSuccess;
}

// Threads a row and chunks a thread.  A row of at most 64 chunks fits one wave (no barrier).  With up to 512 rows the time is one
// row's latency: a chunk a thread (1 x 4096 bf16 5.1 -> 3.7 us, 256 x 8192 12.8 -> 7.3); with more, two and four chunks a thread keep
// more rows on a CU (16384 x 4096: 110 us, 125 with one; 2048 x 8192: 38.1, 42.1 with one).
template <typename T>
hipError_t norm_res_of(const qcnn_norm_res_t &a, hipStream_t s)
{
    const int c = (a.d + Chunk<T>::VE - 1) / Chunk<T>::VE;
    const bool few = a.rows <= 512;
    if (c <= 8) return run<T, 8, 1>(a, s);
    if (c <= 16) return run<T, 16, 1>(a, s);
    if (c <= 32) return run<T, 32, 1>(a, s);
    if (c <= 64) return run<T, 64, 1>(a, s);
    if (c <= 128 && !few) return run<T, 64, 2>(a, s);
    if (c <= 256) return run<T, 256, 1>(a, s);
    if (c <= 512) return few ? run<T, 512, 1>(a, s) : run<T, 256, 2>(a, s);
    if (c <= 1024) return few ? run<T, 1024, 1>(a, s) : run<T, 256, 4>(a, s);
    if (c <= 2048) return run<T, 1024, 2>(a, s);
    if (c <= 4096) return run<T, 1024, 4>(a, s);
    if (c <= 8192) return run<T, 1024, 8>(a, s);
    return run<T, 1024, 16>(a, s);  // float32 rows of up to 65536
}

}  // namespace qcnn
