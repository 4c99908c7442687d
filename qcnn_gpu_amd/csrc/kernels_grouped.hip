// Products grouped by expert (qcnn_op_grouped_matmul): for the rows r of expert e
//   y[r][j] = row_scale[r] * act(w_scale[e][j] * x_scale[s] * sum_k w[e][j][k] * x[s][k] + bias[e][j]),  s = src[r].
#include "block_ops.h"

namespace qcnn {

// 16 bytes of a row are a chunk; a matrix instruction of 16 x 16 outputs takes a chunk of every lane: lane l holds
// chunk (l >> 4) of four of row l & 15.  Both operands come in the same order, so the order of k inside a chunk is free:
// float32 takes four instructions, element i of every lane's chunk each.
template <typename T>
struct Mma {
    typedef f32x4 acc_t;
};
template <>
struct Mma<int8_t> {
    typedef i32x4 acc_t;
};
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mma(f16_t, u32x4 a, u32x4 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(bf16_t, u32x4 a, u32x4 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ i32x4 mma(int8_t, u32x4 a, u32x4 b, i32x4 c)
{
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(float, u32x4 a, u32x4 b, f32x4 c)
{
    const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[i], fb[i], c, 0, 0, 0);
    return c;
}

// The rows of tile `mt` (tiles of TM rows, counted through the experts in turn): expert, first row and row count;
// false beyond the last tile.  A wave does it alone: 64 experts at a time, their tile counts summed up over the lanes.
struct RowTile {
    int e, first, count;
};
__device__ __forceinline__ bool find_tile(const qcnn_grouped_matmul_t &a, int TM, unsigned mt, RowTile &t)
{
    const int lane = threadIdx.x & 63;
    unsigned before = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 64) {
        const int e = e0 + lane;
        int lo = 0, hi = 0;
        if (e < a.experts) {
            lo = min(max(a.offsets[e], 0), a.rows);
            hi = max(min(max(a.offsets[e + 1], 0), a.rows), lo);
        }
        const unsigned tiles = ((unsigned)(hi - lo) + TM - 1) / TM;
        unsigned sum = tiles;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned u = __shfl_up(sum, o);
            if (lane >= o) sum += u;
        }
        const unsigned total = __shfl(sum, 63);
        if (mt < before + total) {
            const unsigned long long mine = __ballot(mt < before + sum);
            const int at = __ffsll(mine) - 1;
            const unsigned start = __shfl(before + sum - tiles, at);
            lo = __shfl(lo, at);
            hi = __shfl(hi, at);
            t.e = __builtin_amdgcn_readfirstlane(e0 + at);
            t.first = __builtin_amdgcn_readfirstlane(lo + (int)(mt - start) * TM);
            t.count = __builtin_amdgcn_readfirstlane(min(TM, hi - lo - (int)(mt - start) * TM));
            return true;
        }
        before += total;
    }
    return false;
}

// Row tiles a call can have: offsets are device memory, so the grid covers the most that `rows` allows; workgroups
// without a tile leave.
static unsigned most_tiles(const qcnn_grouped_matmul_t &a, int TM) { return (unsigned)(a.rows / TM + (a.experts < a.rows ? a.experts : a.rows)); }

// The epilogue of one accumulator (sum) for output j of the expert and row r of y (src row s, `have`: it exists).
struct Epilogue {
    float xs, rs;
    bool have;
    __device__ __forceinline__ void row(const qcnn_grouped_matmul_t &a, int r, int s, bool exists)
    {
        have = exists;
        xs = a.x_scale && exists ? a.x_scale[s] : 1.f;
        rs = a.row_scale ? a.row_scale[r] : 1.f;
    }
    __device__ __forceinline__ float value(const qcnn_grouped_matmul_t &a, float sum, float ws, float b) const
    {
        const float v = have ? sum * ws * xs : 0.f;
        return block_act(v + b, a.act) * rs;
    }
};

typedef u32x4 u32x4_any __attribute__((aligned(1)));
__device__ const u32x4 k_zero_chunk = {0, 0, 0, 0};  // what a lane loads where a row has ended

// Chunk c of a row of `bytes` bytes, at any address; what lies behind the row's end reads as zero.
__device__ __forceinline__ u32x4 load_chunk(const char *row, int c, int bytes)
{
    const int left = bytes - c * 16;
    if (left >= 16) return *(const u32x4_any *)(row + c * 16);
    u32x4 v = {0, 0, 0, 0};
    if (left > 0) {
        unsigned char b[16];
#pragma unroll
        for (int i = 0; i < 15; ++i) b[i] = i < left ? (unsigned char)row[c * 16 + i] : 0;
        b[15] = 0;
        __builtin_memcpy(&v, b, 16);
    }
    return v;
}

// Sixteen bytes from global memory straight into LDS: lane l's go to lds + 16 l.  (m0 is listed as clobbered so that the
// compiler keeps nothing of its own in it; it warns of a reserved register.  The s_nop is the wait state between the
// write of m0 and the load that reads it.)
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(const char *from, unsigned lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(from) : "memory", "m0");
}

// ---- tiles through LDS ---------------------------------------------------------------------------------
// A workgroup of WM x WN waves computes TM rows x TN outputs.  Each step brings 128 bytes of TM rows of x and TN rows of
// w into one of two LDS buffers while the matrix instructions run on the other; a wave owns TM / WM rows x TN / WN
// outputs.  Chunk c of tile row i stands in slot c ^ (i >> 1 & 7) of its row: the sixteen lanes that a ds_read_b128
// serves at a time then touch sixteen different 16-byte slots of the 256 bytes that the banks hold.
// ALIGNED (rows begin at multiples of 16 bytes and hold whole chunks): loads go straight to LDS, a lane whose row
// has ended loads zeros.  Otherwise loads of any address go through registers.
template <typename T, int TM, int TN, int WM, int WN, bool ALIGNED>
__global__ __launch_bounds__(64 * WM *WN, (TM * TN >= 65536 ? 1 : 2)) void k_grouped_tile(const qcnn_grouped_matmul_t a, unsigned nt)
{
    constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
    constexpr int FM = TM / WM / 16, FN = TN / WN / 16;             // 16 x 16 tiles of a wave
    constexpr int LX = TM * 8 / THREADS, LW = TN * 8 / THREADS;     // chunks a thread loads in one step
    constexpr int BUF = (TM + TN) * 128;
    static_assert(LX >= 1 && LW >= 1 && TM * 8 % THREADS == 0 && TN * 8 % THREADS == 0, "whole chunks a thread");
    extern __shared__ __align__(256) char lds[];
    typedef typename Mma<T>::acc_t acc_t;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned mt = blockIdx.x / nt;
    const int n0 = (int)(blockIdx.x % nt) * TN;
    RowTile t;
    if (!find_tile(a, TM, mt, t)) return;

    // this thread's chunks: slot p of tile row i is thread i * 8 + p of a pass; it holds chunk p ^ (i >> 1 & 7)
    const int bytes = a.k * (int)sizeof(T), slot = tid & 7;
    const char *xp[LX], *wp[LW];
    int xc[LX], wc[LW];
#pragma unroll
    for (int i = 0; i < LX; ++i) {
        const int row = (tid + i * THREADS) >> 3;
        const int r = t.first + min(row, t.count - 1);
        const int s = a.src ? a.src[r] : r;
        xp[i] = (const char *)a.x + (size_t)(s >= 0 && s < a.x_rows ? s : 0) * a.ldx * sizeof(T);
        xc[i] = slot ^ (row >> 1 & 7);
    }
#pragma unroll
    for (int i = 0; i < LW; ++i) {
        const int row = (tid + i * THREADS) >> 3;
        wp[i] = (const char *)a.w + ((size_t)t.e * a.w_stride + (size_t)min(n0 + row, a.n - 1) * a.ldw) * sizeof(T);
        wc[i] = slot ^ (row >> 1 & 7);
    }
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char *)lds;
    const int steps = (bytes + 127) / 128;
    u32x4 held[ALIGNED ? 1 : LX + LW];
    const auto request = [&](int step, int buf) {
        if constexpr (ALIGNED) {
            const bool whole = (step + 1) * 128 <= bytes;
            const unsigned at = lds0 + buf * BUF + wave * 1024;
#pragma unroll
            for (int i = 0; i < LX; ++i) {
                const char *p = xp[i] + (size_t)step * 128 + xc[i] * 16;
                if (!whole && step * 128 + xc[i] * 16 >= bytes) p = (const char *)&k_zero_chunk;
                load_to_lds(p, at + i * (THREADS * 16));
            }
#pragma unroll
            for (int i = 0; i < LW; ++i) {
                const char *p = wp[i] + (size_t)step * 128 + wc[i] * 16;
                if (!whole && step * 128 + wc[i] * 16 >= bytes) p = (const char *)&k_zero_chunk;
                load_to_lds(p, at + TM * 128 + i * (THREADS * 16));
            }
        } else {
#pragma unroll
            for (int i = 0; i < LX; ++i) held[i] = load_chunk(xp[i], step * 8 + xc[i], bytes);
#pragma unroll
            for (int i = 0; i < LW; ++i) held[LX + i] = load_chunk(wp[i], step * 8 + wc[i], bytes);
        }
    };
    const auto deposit = [&](int buf) {
        if constexpr (!ALIGNED) {
#pragma unroll
            for (int i = 0; i < LX; ++i) *(u32x4 *)(lds + buf * BUF + (tid + i * THREADS) * 16) = held[i];
#pragma unroll
            for (int i = 0; i < LW; ++i) *(u32x4 *)(lds + buf * BUF + TM * 128 + (tid + i * THREADS) * 16) = held[LX + i];
        }
    };

    const int wm = wave % WM, wn = wave / WM, c16 = lane & 15, g = lane >> 4;
    acc_t acc[FN][FM];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int i = 0; i < FM; ++i) acc[j][i] = acc_t{0, 0, 0, 0};

    request(0, 0);
    deposit(0);
    for (int step = 0; step < steps; ++step) {
        const int buf = step & 1;
        // this step's chunks have landed, here and (after the barrier) everywhere; everyone is done with the other buffer
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (step + 1 < steps) request(step + 1, buf ^ 1);
        const char *bx = lds + buf * BUF + (wm * (TM / WM) + c16) * 128, *bw = lds + buf * BUF + TM * 128 + (wn * (TN / WN) + c16) * 128;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = ((h * 4 + g) ^ (c16 >> 1)) * 16;  // rows of a wave's tiles begin at multiples of 16
            u32x4 fx[FM], fw[FN];
#pragma unroll
            for (int i = 0; i < FM; ++i) fx[i] = *(const u32x4 *)(bx + i * 2048 + at);
#pragma unroll
            for (int j = 0; j < FN; ++j) fw[j] = *(const u32x4 *)(bw + j * 2048 + at);
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int i = 0; i < FM; ++i) acc[j][i] = mma(T(), fw[j], fx[i], acc[j][i]);
        }
        if (step + 1 < steps) deposit(buf ^ 1);
    }

    // lane: row c16 of each row tile, outputs 4 g .. 4 g + 3 of each output tile
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int row = wm * (TM / WM) + i * 16 + c16;
        if (row >= t.count) continue;
        const int r = t.first + row, s = a.src ? a.src[r] : r;
        Epilogue ep;
        ep.row(a, r, s, s >= 0 && s < a.x_rows);
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int n = n0 + wn * (TN / WN) + j * 16 + 4 * g;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (n + q < a.n) {
                    const size_t o = (size_t)t.e * a.n + n + q;
                    const float v = ep.value(a, (float)acc[j][i][q], a.w_scale ? a.w_scale[o] : 1.f, a.bias ? a.bias[o] : 0.f);
                    store_typed(a.y, (size_t)r * a.ldy + n + q, a.out_type, v);
                }
        }
    }
}

template <typename T, int TM, int TN, int WM, int WN>
static hipError_t run_tile(const qcnn_grouped_matmul_t &a, bool al, hipStream_t s)
{
    const unsigned nt = (unsigned)((a.n + TN - 1) / TN);
    const unsigned long long blocks = (unsigned long long)most_tiles(a, TM) * nt;
    if (blocks * (64 * WM * WN) > 0xffffffffull) return hipErrorInvalidConfiguration;
    constexpr int LDS = 2 * (TM + TN) * 128;
    const void *fn = al ? (const void *)k_grouped_tile<T, TM, TN, WM, WN, true> : (const void *)k_grouped_tile<T, TM, TN, WM, WN, false>;
    if (LDS > 65536) {
        const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) return e;
    }
    if (al)
        k_grouped_tile<T, TM, TN, WM, WN, true><<<(unsigned)blocks, 64 * WM * WN, LDS, s>>>(a, nt);
    else
        k_grouped_tile<T, TM, TN, WM, WN, false><<<(unsigned)blocks, 64 * WM * WN, LDS, s>>>(a, nt);
    return hipGetLastError();
}

template <typename T>
static hipError_t pick(qcnn_grouped_matmul_t a, hipStream_t s)
{
    if (a.x_rows == 0) a.x = a.w, a.ldx = 0;  // every row is a row of zeros: what is read is dropped
    const size_t z = sizeof(T);
    const bool al = (uintptr_t)a.x % 16 == 0 && (uintptr_t)a.w % 16 == 0 && a.ldx * z % 16 == 0 && a.ldw * z % 16 == 0 && a.w_stride * z % 16 == 0 &&
                    a.k * z % 16 == 0;
    const long long tiles = (long long)a.rows * a.n / 65536;
    if (tiles >= 256 && al && sizeof(T) < 4) return run_tile<T, 256, 256, 2, 4>(a, al, s);
    return run_tile<T, 128, 128, 2, 2>(a, al, s);
}

hipError_t launch_grouped_matmul(const qcnn_grouped_matmul_t &a, hipStream_t s)
{
    if (a.type == QCNN_F32) return pick<float>(a, s);
    if (a.type == QCNN_F16) return pick<f16_t>(a, s);
    if (a.type == QCNN_BF16) return pick<bf16_t>(a, s);
    return pick<int8_t>(a, s);
}

}  // namespace qcnn
