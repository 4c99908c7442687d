// Products grouped by expert (qcnn_op_grouped_matmul): for the rows r of expert e
//   y[r][j] = row_scale[r] * act(w_scale[e][j] * x_scale[s] * sum_k w[e][j][k] * x[s][k] + bias[e][j]),  s = src[r].
#include "block_ops.h"

#include <type_traits>

namespace qcnn {

// 16 bytes of a row are a chunk; a matrix instruction of 16 x 16 outputs takes a chunk of every lane: lane l holds
// chunk (l >> 4) of four of row l & 15.  Both operands come in the same order, so the order of k inside a chunk is free:
// float32 takes four instructions, element i of every lane's chunk each.
template <typename T>
struct Mma {
    typedef f32x4 acc_t;
    typedef float one_t;
};
template <>
struct Mma<int8_t> {
    typedef i32x4 acc_t;
    typedef int one_t;
};

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

// A tile of TM rows of one expert and TN outputs, or (parts = 2) half of its rows.
struct Tile {
    int e, first, count, n0, parts;
};

// The tiles of a call.  They are counted through the experts in turn; workgroups are dealt to the 8 XCDs round robin
// (blockIdx.x & 7), each with an L2 of its own, so XCD x takes the x-th eighth of the tiles in order, its workgroups one
// after the other, and inside an expert the order walks bands of 8 row tiles column by column: the 32 workgroups that
// run on an XCD at a time then share 8 row tiles of x and 4 column tiles of w.
// The offsets are device memory, so each wave adds up the tiles itself, 64 experts at a time over its lanes.
// PARTS = 2: a tile of at most half of its rows is made as a half, and where the last round of an XCD's workgroups, PER_CU
// on a CU, would leave half of its CUs idle, its tiles are cut in halves (measured as the table at `pick`: 4096 rows over 8, 2048 x 4096
// bfloat16 123 -> 116 us, 16384 over 16, 4096 x 2048 312 -> 308, int8 8192 over 8, 4096 x 4096 184 -> 174; quarters, and halves of
// 64 x 64 tiles, were no faster).
template <int TM, int TN, int PARTS = 1, int PER_CU = 1>
struct Tiles {
    unsigned all, nt;  // row tiles of all experts, column tiles

    static __device__ __forceinline__ unsigned scan(const qcnn_grouped_matmul_t &a, int e0, int &lo, int &hi, unsigned &tiles)
    {
        const int lane = threadIdx.x & 63, e = e0 + lane;
        lo = hi = 0;
        if (e < a.experts) {
            lo = min(max(a.offsets[e], 0), a.rows);
            hi = max(min(max(a.offsets[e + 1], 0), a.rows), lo);
        }
        tiles = ((unsigned)(hi - lo) + TM - 1) / TM;
        unsigned sum = tiles;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned u = __shfl_up(sum, o);
            if (lane >= o) sum += u;
        }
        return sum;
    }
    __device__ __forceinline__ void count(const qcnn_grouped_matmul_t &a)
    {
        nt = ((unsigned)a.n + TN - 1) / TN;
        all = 0;
        for (int e0 = 0; e0 < a.experts; e0 += 64) {
            int l, h;
            unsigned n;
            all += __builtin_amdgcn_readlane(scan(a, e0, l, h, n), 63);
        }
    }
    // the i-th tile of this workgroup's XCD, false beyond the last
    __device__ __forceinline__ bool get(const qcnn_grouped_matmul_t &a, unsigned i, Tile &t) const
    {
        const unsigned per = (all * nt + 7) / 8;
        unsigned piece = 0, pieces = 1;
        if constexpr (PARTS > 1) {
            const unsigned walkers = gridDim.x >> 3, whole = per / walkers * walkers, left = per - whole;
            if (i >= whole) {
                pieces = left * PARTS * PER_CU > walkers ? 1 : PARTS;
                piece = (i - whole) % pieces;
                i = whole + (i - whole) / pieces;
            }
        }
        const unsigned at = (blockIdx.x & 7) * per + i;
        if (i >= per || at >= all * nt) return false;
        int l0, h0, e0 = 0;
        unsigned n, s = scan(a, 0, l0, h0, n), before = 0;
        for (;;) {
            const unsigned total = __builtin_amdgcn_readlane(s, 63);
            if (at < (before + total) * nt) break;
            before += total;
            e0 += 64;
            if (e0 >= a.experts) return false;
            s = scan(a, e0, l0, h0, n);
        }
        const unsigned long long at_or_behind = __ballot(at < (before + s) * nt);
        if (!at_or_behind) return false;
        const int l = __ffsll(at_or_behind) - 1;
        const unsigned m = __builtin_amdgcn_readlane(n, l), in = at - (before + __builtin_amdgcn_readlane(s, l) - m) * nt;
        // Offsets that decrease can make more tiles than the grid was made for, and sums that wrap: what does not lie in the
        // expert found is dropped (m * nt < 2^32, the host has seen to it).
        if (in >= m * nt) return false;
        const unsigned band = in / (8 * nt), rows = min(8u, m - band * 8), rest = in - band * 8 * nt;
        t.e = e0 + l;
        t.first = __builtin_amdgcn_readlane(l0, l) + (int)(band * 8 + rest % rows) * TM + (int)(piece * (TM / pieces));
        t.count = min((int)(TM / pieces), (int)__builtin_amdgcn_readlane(h0, l) - t.first);
        t.n0 = (int)(rest / rows) * TN;
        t.parts = t.count <= TM / PARTS ? PARTS : 1;
        return t.count > 0;  // (a part without rows: of the last round)
    }
};

// Row tiles a call can have: offsets are device memory, so the grid covers the most that `rows` allows (each expert
// with rows ends in one short tile); workgroups without a tile leave.  `tiles` stays below 2^31, n below 2^28.
static hipError_t count_tiles(const qcnn_grouped_matmul_t &a, int TM, int TN, unsigned long long &tiles)
{
    tiles = ((unsigned long long)(a.rows / TM) + (a.experts < a.rows ? a.experts : a.rows)) * ((a.n + TN - 1) / TN);
    return tiles < 1ull << 31 ? hipSuccess : hipErrorNotSupported;
}

// N neighbouring outputs of one row.  `least` is 0 for ReLU, else -inf (a NaN passes either way).  STREAM: past the caches.
template <typename OT, int N, bool STREAM = false>
__device__ __forceinline__ void store_row(const qcnn_grouped_matmul_t &a, const float (&v)[N], float rs, float least, size_t r, int n)
{
    OT o[N];
#pragma unroll
    for (int q = 0; q < N; ++q) from_f32((v[q] < least ? least : v[q]) * rs, o[q]);
    OT *y = (OT *)a.y + r * a.ldy + n;
    if (n + N <= a.n) {
        constexpr int C = sizeof o / 16;
        u32x4 c[C];
        __builtin_memcpy(c, o, sizeof o);
#pragma unroll
        for (int i = 0; i < C; ++i) {
            if constexpr (STREAM)
                __builtin_nontemporal_store(c[i], (u32x4_any *)y + i);
            else
                ((u32x4_any *)y)[i] = c[i];
        }
    } else {
#pragma unroll
        for (int q = 0; q < N - 1; ++q)
            if (n + q < a.n) y[q] = o[q];
    }
}

// Outputs of an expert stand in its tiles in another order than in memory: of 32 of them, output 8 g + 4 h + q is row
// 4 g + q of 16 x 16 tile h.  The lane that holds rows 4 g .. 4 g + 3 of both tiles then has eight neighbouring outputs,
// 16 bytes of a half row, and four lanes 64 bytes of y (with 8 bytes a lane the stores of a 256 x 256 tile took 20 us, a
// quarter of the time of 2048 k).
__device__ __forceinline__ int output_at(int row) { return (row & ~31) | (row >> 2 & 3) << 3 | (row >> 4 & 1) << 2 | (row & 3); }

// The epilogue of a wave's FN x FM accumulators of 16 outputs x 16 rows: the lane has outputs n0 .. n0 + 7 (of each pair
// of output tiles, 32 further on) of row row0 of each row tile (16 further on); `count` rows of the tile exist.
template <int FN, int FM, typename A>
__device__ __forceinline__ void epilogue(const qcnn_grouped_matmul_t &a, const A (&acc)[FN][FM], int e, int first, int row0, int count, int n0)
{
    static_assert(FN % 2 == 0, "pairs of output tiles");
    const float least = a.act == QCNN_ACT_RELU ? 0.f : -__builtin_inff();
    float xs[FM], rs[FM];
    bool have[FM];
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int row = row0 + i * 16, r = first + min(row, count - 1), s = a.src ? a.src[r] : r;
        have[i] = s >= 0 && s < a.x_rows;  // of another row what was summed up is dropped
        xs[i] = a.x_scale && have[i] ? a.x_scale[s] : 1.f;
        rs[i] = a.row_scale ? a.row_scale[r] : 1.f;
    }
    const auto all = [&](auto type) {
        typedef decltype(type) OT;
#pragma unroll
        for (int j = 0; j < FN; j += 2) {
            const int n = n0 + j * 16;
            if (n >= a.n) continue;
            float ws[8], b[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) ws[q] = 1.f, b[q] = 0.f;
            if (a.w_scale) {
#pragma unroll
                for (int q = 0; q < 8; ++q) ws[q] = a.w_scale[(size_t)e * a.n + min(n + q, a.n - 1)];
            }
            if (a.bias) {
#pragma unroll
                for (int q = 0; q < 8; ++q) b[q] = a.bias[(size_t)e * a.n + min(n + q, a.n - 1)];
            }
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                float v[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) v[q] = (have[i] ? (float)acc[j + (q >> 2)][i][q & 3] * ws[q] * xs[i] : 0.f) + b[q];
                if (a.act == QCNN_ACT_SILU) {
#pragma unroll
                    for (int q = 0; q < 8; ++q) v[q] = block_act(v[q], QCNN_ACT_SILU);
                }
                if (row0 + i * 16 < count) store_row<OT>(a, v, rs[i], least, (size_t)(first + row0 + i * 16), n);
            }
        }
    };
    if (a.out_type == QCNN_F32)
        all(float());
    else if (a.out_type == QCNN_F16)
        all(f16_t());
    else
        all(bf16_t());
}

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
// A workgroup of WM x WN waves computes TM rows x TN outputs, a wave TM / WM x TN / WN of them.  A step is 64 bytes of k:
// its chunks of TM rows of x and TN rows of w go into one of four LDS buffers, requested four steps before the matrix
// instructions use them and read into registers one step before: in step s the instructions run on registers, s + 1 is
// read from LDS, s + 2 and s + 3 are on their way and s + 4 is requested into the buffer that s left.  One barrier a step.
// Chunk c of tile row i stands in slot c ^ f of the row's four, f = 0, 0, 3, 3 for (i >> 2 & 3): the sixteen lanes that a
// ds_read_b128 serves at a time (rows 0-3 and 12-15 of one chunk, 4-11 of the next) then touch sixteen different slots
// of the 256 bytes that the banks hold.
// ALIGNED (rows begin at multiples of 16 bytes and hold whole chunks): loads go straight to LDS, a lane whose row
// has ended loads zeros.  Otherwise loads of any address go through registers, a step ahead of LDS.
// Measured with tiles of 256 x 256, one expert: 8192 x 8192 x 8192 1260 TFLOP/s in bfloat16 (the library's product 1330 to 1375)
// and 2280 TOP/s in int8; 16384 rows over 16, 4096 x 2048: 300 to 308 us, 890 to 916 TFLOP/s: short last tiles, the last round and the
// hand-over between tiles, a chain of waits, take the rest.
template <int TM, int TN, int WM, int WN>
struct TileGeom {
    static constexpr int LDS = 4 * (TM + TN) * 64, PER_CU = 163840 / LDS < 8 / (WM * WN) ? 163840 / LDS : 8 / (WM * WN);
    static constexpr int PARTS = TM >= 128 ? 2 : 1;
};

template <typename T, int TM, int TN, int WM, int WN, bool ALIGNED>
__global__ __launch_bounds__(64 * WM *WN, 2) void k_grouped_tile(const qcnn_grouped_matmul_t a)
{
    constexpr int WAVES = WM * WN, THREADS = 64 * WAVES, PARTS = TileGeom<TM, TN, WM, WN>::PARTS;
    constexpr int FM = TM / WM / 16, FN = TN / WN / 16;             // 16 x 16 tiles of a wave
    constexpr int LX = TM * 4 / THREADS, LW = TN * 4 / THREADS;     // chunks a thread loads in one step
    constexpr int BUF = (TM + TN) * 64;
    static_assert(LX >= 1 && LW >= 1 && TM * 4 % THREADS == 0 && TN * 4 % THREADS == 0, "whole chunks a thread");
    extern __shared__ __align__(256) char lds[];
    typedef typename Mma<T>::acc_t acc_t;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Tiles<TM, TN, PARTS, TileGeom<TM, TN, WM, WN>::PER_CU> tiles;
    tiles.count(a);
    Tile t{0, 0, 0, 0, 1}, next_t;
    unsigned index = blockIdx.x >> 3;
    if (!tiles.get(a, index, t)) return;

    const int bytes = a.k * (int)sizeof(T);
    const auto swizzle = [](int row) { return (row >> 3 & 1) * 3; };
    const char *xp[LX], *wp[LW];  // the rows of which this thread brings a chunk a step
    static_assert(THREADS % 64 == 0, "all of a thread's chunks stand in the same slot of their rows");
    const int chunk = ((tid & 3) ^ swizzle(tid >> 2)) * 16;
    const auto rows_of = [&](const Tile &t) {
#pragma unroll
        for (int i = 0; i < LX; ++i) {
            const int r = t.first + min((tid + i * THREADS) >> 2, t.count - 1);
            const int s = a.src ? a.src[r] : r;
            xp[i] = (const char *)a.x + (size_t)(s >= 0 && s < a.x_rows ? s : 0) * a.ldx * sizeof(T) + (ALIGNED ? chunk : 0);
        }
#pragma unroll
        for (int i = 0; i < LW; ++i)
            wp[i] = (const char *)a.w + ((size_t)t.e * a.w_stride + (size_t)min(t.n0 + output_at((tid + i * THREADS) >> 2), a.n - 1) * a.ldw) * sizeof(T) +
                    (ALIGNED ? chunk : 0);
    };
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char *)lds;
    const int steps = (bytes + 63) / 64;
    u32x4 held[ALIGNED ? 1 : LX + LW];
    // asks for chunk i of the thread's lx + LW of a step; called step after step, the pointers walk
    const auto request_one = [&](int lx, int step, int i, bool ended) {
        const char *&p = i < lx ? xp[i < lx ? i : 0] : wp[i < lx ? 0 : i - lx];
        const unsigned at = lds0 + (step & 3) * BUF + wave * 1024 + (i < lx ? i * (THREADS * 16) : TM * 64 + (i - lx) * (THREADS * 16));
        load_to_lds(ended ? (const char *)&k_zero_chunk : p, at);
        p += 64;
    };
    const auto request = [&](auto lx, int step) {
        if constexpr (ALIGNED) {
            const bool ended = step * 64 + chunk >= bytes;
#pragma unroll
            for (int i = 0; i < lx() + LW; ++i) request_one(lx(), step, i, ended);
        } else {
#pragma unroll
            for (int i = 0; i < lx(); ++i) held[i] = load_chunk(xp[i], step * 4 + chunk / 16, bytes);
#pragma unroll
            for (int i = 0; i < LW; ++i) held[LX + i] = load_chunk(wp[i], step * 4 + chunk / 16, bytes);
        }
    };
    const auto deposit = [&](auto lx, int step) {
        if constexpr (!ALIGNED) {
            char *at = lds + (step & 3) * BUF + tid * 16;
#pragma unroll
            for (int i = 0; i < lx(); ++i) *(u32x4 *)(at + i * (THREADS * 16)) = held[i];
#pragma unroll
            for (int i = 0; i < LW; ++i) *(u32x4 *)(at + TM * 64 + i * (THREADS * 16)) = held[LX + i];
        }
    };

    const int wm = wave % WM, wn = wave / WM, c16 = lane & 15, g = lane >> 4;
    const int from = c16 * 64 + (g ^ swizzle(c16)) * 16;  // rows of a wave's tiles begin at multiples of 16
    const auto with_parts = [&](int parts, auto f) {
        parts = __builtin_amdgcn_readfirstlane(parts);
        if constexpr (PARTS > 1) {
            if (parts == PARTS) return f(std::integral_constant<int, PARTS>());
        }
        f(std::integral_constant<int, 1>());
    };
    // chunks of x that a thread asks for in one step, at least one: those of rows that do not count are the last row's
    const auto chunks_of = [](auto parts) { return std::integral_constant<int, (LX / parts() > 0 ? LX / parts() : 1)>(); };

    const auto begin = [&](auto lx) {
        request(lx, 0);
        if constexpr (ALIGNED) {
            if (1 < steps) request(lx, 1);
            if (2 < steps) request(lx, 2);
        }
    };
    rows_of(t);
    with_parts(t.parts, [&](auto p) { begin(chunks_of(p)); });
    bool more = false;
    const auto product = [&](auto parts) {
        constexpr int M = FM / parts(), L = decltype(chunks_of(parts))::value;
        constexpr std::integral_constant<int, L> lx;
        u32x4 fw[FN], fx[2][M];  // a step's operands; w of the next step takes the place of what has been used
        const auto read_w = [&](int step, int j) { fw[j] = *(const u32x4 *)(lds + (step & 3) * BUF + from + TM * 64 + wn * (TN / WN) * 64 + j * 1024); };
        const auto read_x = [&](int step, u32x4(&x)[M], int i) { x[i] = *(const u32x4 *)(lds + (step & 3) * BUF + from + wm * (M * 16) * 64 + i * 1024); };
        const auto read = [&](int step) {
#pragma unroll
            for (int j = 0; j < FN; ++j) read_w(step, j);
#pragma unroll
            for (int i = 0; i < M; ++i) read_x(step, fx[0], i);
        };
        acc_t acc[FN][M];
        const auto multiply_part = [&](const u32x4(&x)[M], int j) {
#pragma unroll
            for (int i = 0; i < M; ++i) acc[j][i] = mma(T(), fw[j], x[i], acc[j][i]);
        };
        const auto multiply = [&](const u32x4(&x)[M]) {
#pragma unroll
            for (int j = 0; j < FN; ++j) multiply_part(x, j);
        };
        // (ALIGNED) The chunks of step s have landed, here and (after the barrier) everywhere, and everyone has read step s - 1
        // into registers.  Loads land in order, so all but those of the two steps behind s are waited for.
        const auto arrive = [&](int s) {
            if (s + 2 < steps)
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * (L + LW)) : "memory");
            else if (s + 1 < steps)
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(L + LW) : "memory");
            else
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        };

#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int i = 0; i < M; ++i) acc[j][i] = acc_t{0, 0, 0, 0};
        if constexpr (ALIGNED) {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (3 < steps) request(lx, 3);
            read(0);
            // Matrix instructions first: their operands are there.  The reads of the next step and the requests stand between
            // groups of them, as a wave issues in order and would hold its matrix instructions up behind them: all of them in
            // front left the matrix cores idle half of the time.  No branch in here; the last steps are made below.
            const auto step = [&](int s, u32x4(&now)[M], u32x4(&next)[M]) {
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * (L + LW)) : "memory");
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    multiply_part(now, j);
                    __builtin_amdgcn_sched_barrier(0);
                    read_w(s + 1, j);
#pragma unroll
                    for (int i = M * j / FN; i < M * (j + 1) / FN; ++i) read_x(s + 1, next, i);
#pragma unroll
                    for (int i = (L + LW) * j / FN; i < (L + LW) * (j + 1) / FN; ++i) request_one(L, s + 4, i, false);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            int s = 0;
            for (; (s + 6) * 64 <= bytes; s += 2) {
                step(s, fx[0], fx[1]);
                step(s + 1, fx[1], fx[0]);
            }
#pragma unroll 1
            for (; s < steps; ++s) {
                multiply(fx[0]);
                if (s + 1 < steps) {
                    arrive(s + 1);
                    if (s + 4 < steps) request(lx, s + 4);
                    read(s + 1);
                }
            }
        } else {
            // Step s: s + 1 is in LDS, s + 2 is put there and s + 3 asked for, behind the matrix instructions of s.
            deposit(lx, 0);
            if (1 < steps) request(lx, 1);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            read(0);
            if (1 < steps) deposit(lx, 1);
            if (2 < steps) request(lx, 2);
#pragma unroll 1
            for (int s = 0; s < steps; ++s) {
                if (s + 1 < steps) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                multiply(fx[0]);
                __builtin_amdgcn_sched_barrier(0);
                if (s + 1 < steps) read(s + 1);
                if (s + 2 < steps) deposit(lx, s + 2);
                if (s + 3 < steps) request(lx, s + 3);
            }
        }
        // the next tile's first chunks are on their way while this one's outputs are written
        index += gridDim.x >> 3;
        more = tiles.get(a, index, next_t);
        if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // everyone has read this tile's last chunks
            rows_of(next_t);
            with_parts(next_t.parts, [&](auto p) { begin(chunks_of(p)); });
        }
        // lane: row c16 of each row tile, outputs 8 g .. 8 g + 7 of each pair of output tiles
        epilogue(a, acc, t.e, t.first, wm * (M * 16) + c16, t.count, t.n0 + wn * (TN / WN) + 8 * g);
    };
    for (;;) {
        with_parts(t.parts, product);
        if (!more) break;
        t = next_t;
    }
}

// ---- few rows an expert --------------------------------------------------------------------------------
// Reading the weights is the cost.  A workgroup takes up to 16 MT rows of one expert and 16 NW outputs; its waves are
// KW x NW, NW share out the outputs and KW the k, in runs of RB bytes, and the KW sums meet in LDS at the end.  Direct loads
// bring the chunks in the order of the matrix instruction's lanes, R - 1 runs ahead: 1 KB of LDS is one operand, 64 bytes of
// k of 16 rows.  x is shared by the NW waves of a k group (one barrier a run, none for NW = 1), and of sixteen rows
// only those that there are ask for it.  64 rows of 64 experts, 1024 x 2048 bfloat16, cold: 38 to 40 us, 4.1 to 4.3 TB/s.
template <typename T, int MT, int RB, int KW, int NW, int KB>
struct RowsGeom {
    static constexpr int OPS = RB / 64, WAVES = KW * NW;
    static constexpr int XB = MT * OPS * 1024, RUN = XB + NW * OPS * 1024;
    static constexpr int XL = MT * OPS / NW, LOADS = OPS + XL;  // direct loads of a wave for one run
    static constexpr int FIT = KB * 1024 / (KW * RUN), R = FIT < 2 ? 2 : FIT < 8 ? FIT : 8;  // runs in the ring: as many as KB kilobytes hold
    static constexpr int SUMS = WAVES * MT * 1024;
    static constexpr int LDS = KW * R * RUN > SUMS ? KW * R * RUN : SUMS;
    static_assert(MT * OPS % NW == 0 && LOADS * (R - 2) < 64 && LDS <= 163840, "runs fit");
};

template <typename T, int MT, int RB, int KW, int NW, int KB, bool ALIGNED>
__global__ __launch_bounds__(64 * KW *NW) void k_grouped_rows(const qcnn_grouped_matmul_t a)
{
    typedef RowsGeom<T, MT, RB, KW, NW, KB> G;
    typedef typename Mma<T>::acc_t acc_t;
    typedef typename Mma<T>::one_t one_t;
    constexpr int OPS = G::OPS, R = G::R;
    extern __shared__ __align__(1024) char lds[];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c16 = lane & 15, g = lane >> 4;
    const int kq = wave / NW, nq = wave % NW;
    Tiles<16 * MT, 16 * NW> tiles;
    tiles.count(a);
    Tile t{0, 0, 0, 0, 1};
    if (!tiles.get(a, workgroup() >> 3, t)) return;

    // this lane's rows: one of w and, for each operand of x that this wave brings, one of x
    const int bytes = a.k * (int)sizeof(T), all = (bytes + RB - 1) / RB, turns = (all + KW - 1) / KW;
    const int first = kq * turns, count = max(0, min(turns, all - first));
    const char *wp = (const char *)a.w + ((size_t)t.e * a.w_stride + (size_t)min(t.n0 + nq * 16 + c16, a.n - 1) * a.ldw) * sizeof(T) + (size_t)first * RB;
    const char *xp[G::XL];
    bool has[G::XL];
#pragma unroll
    for (int i = 0; i < G::XL; ++i) {
        const int row = (i * NW + nq) / OPS * 16 + c16, r = t.first + min(row, t.count - 1), s = a.src ? a.src[r] : r;
        has[i] = MT > 1 || row < t.count;  // (a load that no lane asks for would not be counted by the waits: one tile always has a row)
        xp[i] = (const char *)a.x + (size_t)(s >= 0 && s < a.x_rows ? s : 0) * a.ldx * sizeof(T) + (size_t)first * RB;
    }
    char *const ring = lds + kq * (R * G::RUN);
    const unsigned ring_at = (unsigned)(size_t)(__attribute__((address_space(3))) char *)ring;
    int bring_slot = 0;
    u32x4 held[ALIGNED ? 1 : OPS + G::XL];
    // brings run i (of this group) into the ring, or (not ALIGNED) into registers; called for 0, 1, 2 ...
    const auto bring = [&](int i) {
        if (i < count) {
            const int left = bytes - (first + i) * RB - g * 16;  // bytes of the rows from this lane's first chunk on
            if constexpr (ALIGNED) {
                const unsigned at = ring_at + bring_slot;
#pragma unroll
                for (int o = 0; o < OPS; ++o) load_to_lds(o * 64 < left ? wp + o * 64 : (const char *)&k_zero_chunk, at + G::XB + (nq * OPS + o) * 1024);
#pragma unroll
                for (int j = 0; j < G::XL; ++j) {
                    const int o = (j * NW + nq) % OPS;
                    if (has[j]) load_to_lds(o * 64 < left ? xp[j] + o * 64 : (const char *)&k_zero_chunk, at + (j * NW + nq) * 1024);
                }
            } else {
#pragma unroll
                for (int o = 0; o < OPS; ++o) held[o] = load_chunk(wp, o * 4, left);
#pragma unroll
                for (int j = 0; j < G::XL; ++j) held[OPS + j] = load_chunk(xp[j], (j * NW + nq) % OPS * 4, left);
            }
            wp += RB;
#pragma unroll
            for (int j = 0; j < G::XL; ++j) xp[j] += RB;
        }
        if constexpr (ALIGNED) bring_slot = bring_slot == (R - 1) * G::RUN ? 0 : bring_slot + G::RUN;
    };
    const auto deposit = [&](int i) {  // run i, from registers
        if constexpr (!ALIGNED) {
            if (i < count) {
                char *at = ring + bring_slot + lane * 16;
#pragma unroll
                for (int o = 0; o < OPS; ++o) *(u32x4 *)(at + G::XB + (nq * OPS + o) * 1024) = held[o];
#pragma unroll
                for (int j = 0; j < G::XL; ++j) *(u32x4 *)(at + (j * NW + nq) * 1024) = held[OPS + j];
            }
            bring_slot = bring_slot == (R - 1) * G::RUN ? 0 : bring_slot + G::RUN;
        }
    };
    wp += g * 16;
#pragma unroll
    for (int j = 0; j < G::XL; ++j) xp[j] += g * 16;

    acc_t acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = acc_t{0, 0, 0, 0};
    int slot = 0;
    if constexpr (ALIGNED) {
#pragma unroll 1
        for (int i = 0; i < R - 1; ++i) bring(i);
    } else {
        bring(0);
        deposit(0);
        bring(1);
    }
    for (int i = 0; i < turns; ++i) {
        // run i has landed (loads land in order: all but those of the runs behind it), here and after the barrier for all, and
        // everyone is done with run i - 1, whose place run i + R - 1 takes (not ALIGNED: run i + 1, from registers; R >= 2)
        if constexpr (ALIGNED)
            wait_for_all_but<R - 2, G::LOADS>(count - 1 - i);
        else
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (NW > 1) asm volatile("s_barrier" ::: "memory");
        if constexpr (ALIGNED) {
            bring(i + R - 1);
        } else {
            deposit(i + 1);
            bring(i + 2);
        }
        if (i < count) {
            const char *at = ring + slot + lane * 16;
            u32x4 w[OPS], x[OPS][MT];
#pragma unroll
            for (int o = 0; o < OPS; ++o) {
                w[o] = *(const u32x4 *)(at + G::XB + (nq * OPS + o) * 1024);
#pragma unroll
                for (int m = 0; m < MT; ++m) x[o][m] = *(const u32x4 *)(at + (m * OPS + o) * 1024);
            }
#pragma unroll
            for (int o = 0; o < OPS; ++o)
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[m] = mma(T(), x[o][m], w[o], acc[m]);
        }
        slot = slot == (R - 1) * G::RUN ? 0 : slot + G::RUN;
    }

    // the k groups' sums; the lane has rows 4 g .. 4 g + 3 of output c16
    __syncthreads();
    one_t *sums = (one_t *)lds;
    constexpr int OUT = 16 * NW;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int q = 0; q < 4; ++q) sums[kq * (OUT * 16 * MT) + (m * 16 + 4 * g + q) * OUT + nq * 16 + c16] = acc[m][q];
    __syncthreads();
    for (int o = threadIdx.x; o < OUT * t.count; o += 64 * KW * NW) {
        const int row = o / OUT, n = t.n0 + o % OUT;
        if (n >= a.n) continue;
        one_t v = 0;
#pragma unroll
        for (int k = 0; k < KW; ++k) v += sums[k * (OUT * 16 * MT) + o];
        const int r = t.first + row, s = a.src ? a.src[r] : r;
        const size_t e = (size_t)t.e * a.n + n;
        float f = 0.f;
        if (s >= 0 && s < a.x_rows) {  // of another row what was summed up is dropped
            f = (float)v;
            if (a.w_scale) f *= a.w_scale[e];
            if (a.x_scale) f *= a.x_scale[s];
        }
        if (a.bias) f += a.bias[e];
        f = block_act(f, a.act);
        if (a.row_scale) f *= a.row_scale[r];
        store_typed(a.y, (size_t)r * a.ldy + n, a.out_type, f);
    }
}

template <typename T, int MT, int RB, int KW, int NW, int KB>
static hipError_t run_rows(const qcnn_grouped_matmul_t &a, bool al, hipStream_t s)
{
    typedef RowsGeom<T, MT, RB, KW, NW, KB> G;
    unsigned long long tiles;
    hipError_t e = count_tiles(a, 16 * MT, 16 * NW, tiles);
    if (e != hipSuccess) return e;
    const unsigned long long blocks = (tiles + 7) / 8 * 8;  // as many on each XCD
    dim3 grid;
    e = grid_of(blocks, grid);
    if (e != hipSuccess) return e;
    static std::atomic<unsigned long long> asked[2] = {{0}, {0}};
    const auto fn = al ? k_grouped_rows<T, MT, RB, KW, NW, KB, true> : k_grouped_rows<T, MT, RB, KW, NW, KB, false>;
    e = allow_lds((const void *)fn, G::LDS, asked[al]);
    if (e != hipSuccess) return e;
    fn<<<grid, 64 * KW * NW, G::LDS, s>>>(a);
    return hipGetLastError();
}

// Compute units of the current device, asked for once.
static int compute_units()
{
    static const int n = [] {
        int dev = 0, cu = 0;
        if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&cu, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cu < 8) cu = 256;
        return cu;
    }();
    return n;
}

template <typename T, int TM, int TN, int WM, int WN>
static hipError_t run_tile(const qcnn_grouped_matmul_t &a, bool al, hipStream_t s)
{
    typedef TileGeom<TM, TN, WM, WN> G;
    unsigned long long tiles;
    hipError_t e = count_tiles(a, TM, TN, tiles);
    if (e != hipSuccess) return e;
    const unsigned long long fit = (unsigned long long)compute_units() * G::PER_CU;
    const unsigned blocks = (unsigned)(((tiles * G::PARTS < fit ? tiles * G::PARTS : fit) + 7) / 8 * 8);  // as many on each XCD; they walk the tiles
    auto fn = k_grouped_tile<T, TM, TN, WM, WN, true>;
    if constexpr (TM < 256) {  // (the largest tiles have no registers for loads of any address)
        if (!al) fn = k_grouped_tile<T, TM, TN, WM, WN, false>;
    }
    static std::atomic<unsigned long long> asked[2] = {{0}, {0}};
    e = allow_lds((const void *)fn, G::LDS, asked[al]);
    if (e != hipSuccess) return e;
    fn<<<blocks, 64 * WM * WN, G::LDS, s>>>(a);
    return hipGetLastError();
}

// ---- short rows and few outputs, many rows ---------------------------------------------------------------
// Up to 64 outputs of rows of up to 256 bytes, the 1x1 layers of an image network: reading x and writing y is the cost.
// A wave keeps the weights of all outputs in registers and runs over its rows, four tiles of sixteen at a time, straight
// from memory into matrix instructions.  Outputs of two bytes stand in the tiles as output_at has them, so that a lane
// has 16 bytes of a row either way and four lanes write 64 side by side, past the caches, which the output would only
// wash out (798720 rows, 48 int8 to 32 float32: 33.4 us where the last cache holds x, 46.6 through them; with cold x 53, and
// 46.6 through them).
template <typename T, int NT, int OPS, int TM>
__global__ __launch_bounds__(256) void k_grouped_narrow(const qcnn_grouped_matmul_t a)
{
    typedef typename Mma<T>::acc_t acc_t;
    constexpr int BATCH = TM == 64 ? 1 : OPS == 1 ? 4 : 2;  // row tiles on their way at a time
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c16 = lane & 15, g = lane >> 4;
    Tiles<TM, 64> tiles;
    tiles.count(a);
    Tile t{0, 0, 0, 0, 1};
    if (!tiles.get(a, workgroup() >> 3, t)) return;

    const int bytes = a.k * (int)sizeof(T);
    const bool pairs = a.out_type != QCNN_F32;
    u32x4 w[NT][OPS];
    f32x4 ws[NT], b[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const char *row = (const char *)a.w + ((size_t)t.e * a.w_stride + (size_t)min(pairs ? output_at(j * 16 + c16) : j * 16 + c16, a.n - 1) * a.ldw) * sizeof(T);
#pragma unroll
        for (int o = 0; o < OPS; ++o) w[j][o] = load_chunk(row, o * 4 + g, bytes);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const size_t n = (size_t)t.e * a.n + min((pairs ? output_at(j * 16 + 4 * g) : j * 16 + 4 * g) + q, a.n - 1);
            ws[j][q] = a.w_scale ? a.w_scale[n] : 1.f;
            b[j][q] = a.bias ? a.bias[n] : 0.f;
        }
    }
    const auto rows = [&](auto type) {
        typedef decltype(type) OT;
        const float least = a.act == QCNN_ACT_RELU ? 0.f : -__builtin_inff();
        for (int m0 = wave * (TM / 4); m0 < min((wave + 1) * (TM / 4), t.count); m0 += 16 * BATCH) {
            u32x4 x[BATCH][OPS];
            float xs[BATCH], rs[BATCH];
            bool have[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int r = t.first + min(m0 + i * 16 + c16, t.count - 1), s = a.src ? a.src[r] : r;
                have[i] = s >= 0 && s < a.x_rows;
                const char *row = (const char *)a.x + (size_t)(have[i] ? s : 0) * a.ldx * sizeof(T);
#pragma unroll
                for (int o = 0; o < OPS; ++o) x[i][o] = load_chunk(row, o * 4 + g, bytes);
                xs[i] = a.x_scale && have[i] ? a.x_scale[s] : 1.f;
                rs[i] = a.row_scale ? a.row_scale[r] : 1.f;
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int m = m0 + i * 16 + c16;
                constexpr int N = 16 / sizeof(OT), TILES = N / 4;  // outputs side by side, of so many tiles
#pragma unroll
                for (int j = 0; j < NT; j += TILES) {
                    float v[N];
#pragma unroll
                    for (int h = 0; h < TILES; ++h) {
                        acc_t acc = {0, 0, 0, 0};
#pragma unroll
                        for (int o = 0; o < OPS; ++o) acc = mma(T(), w[j + h][o], x[i][o], acc);
#pragma unroll
                        for (int q = 0; q < 4; ++q) v[4 * h + q] = (have[i] ? (float)acc[q] * ws[j + h][q] * xs[i] : 0.f) + b[j + h][q];
                    }
                    if (a.act == QCNN_ACT_SILU) {
#pragma unroll
                        for (int q = 0; q < N; ++q) v[q] = block_act(v[q], QCNN_ACT_SILU);
                    }
                    const int n = j * 16 + N * g;
                    if (m < t.count && n < a.n) store_row<OT, N, true>(a, v, rs[i], least, (size_t)(t.first + m), n);
                }
            }
        }
    };
    if (a.out_type == QCNN_F32)
        rows(float());
    else if (a.out_type == QCNN_F16)
        rows(f16_t());
    else
        rows(bf16_t());
}

template <typename T, int NT, int OPS, int TM>
static hipError_t launch_narrow(const qcnn_grouped_matmul_t &a, hipStream_t s)
{
    unsigned long long tiles;
    hipError_t e = count_tiles(a, TM, 64, tiles);
    if (e != hipSuccess) return e;
    dim3 grid;
    e = grid_of((tiles + 7) / 8 * 8, grid);
    if (e != hipSuccess) return e;
    k_grouped_narrow<T, NT, OPS, TM><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

// 512 rows a workgroup where that makes enough of them, else 64 (3968 rows of 209 bytes 25 -> 9.8 us).
template <typename T, int NT, int OPS>
static hipError_t run_narrow(const qcnn_grouped_matmul_t &a, hipStream_t s)
{
    return a.rows >= 131072 ? launch_narrow<T, NT, OPS, 512>(a, s) : launch_narrow<T, NT, OPS, 64>(a, s);
}

template <typename T>
static hipError_t pick(qcnn_grouped_matmul_t a, hipStream_t s)
{
    if (a.x_rows == 0) a.x = a.w, a.ldx = 0;  // every row is a row of zeros: what is read is dropped
    const size_t z = sizeof(T);
    const bool al = (uintptr_t)a.x % 16 == 0 && (uintptr_t)a.w % 16 == 0 && a.ldx * z % 16 == 0 && a.ldw * z % 16 == 0 && a.w_stride * z % 16 == 0 &&
                    a.k * z % 16 == 0;
    // Which kernel, by the rows an expert has on average (the host does not know the offsets) and the tiles there can be.
    // Microseconds of the taken side and of the other: a call of a captured graph of calls, median of 9, inputs cold (copies of the
    // buffers in turn), skewed loads, rows gathered and scaled, bias and ReLU (lines marked *: the cases of perf/operators.py);
    // bfloat16 where no type is named:
    //   narrow    798720 rows 48 -> 32 int8 *          53, tiles 76
    //   rows      64 over 64 experts, 1024 x 2048 *    39, 128 x 128 tiles 51;  7 rows 157 x 3840: 8 k groups 8.5, 4 11.8
    //             128 over 16, 2048 x 2048             34, 16 rows a workgroup 37;  200 over 8, 300 x 1000: 9.6, 64 x 64 tiles 12.2
    //             float32 400 over 8, 300 x 2001       24, 64 x 64 tiles 124;  500 of one, 900 x 1024: 22, 64 x 64 24
    //   64 x 64   1024 over 16, 1024 x 1024            19, 128 x 128 20;  512 over 4, 1024 x 1024: 12.1, rows 21
    //             float32 5000 over 5, 1000 x 2000    200, 128 x 128 253
    //             float32 1000 of one, 800 x 1000      25, rows 36
    //   128 x 128 8900 over 22, 1424 x 1944           131, 256 x 256 146;  8192 over 64, 2048 x 2048: 167, 256 x 256 186
    //             short k: 16384 over 8, 1024 x 512     41, 256 x 256 43;  int8 8192 over 16, 2048 x 1024: 47, 256 x 256 48
    //   256 x 256 16384 over 16, 4096 x 2048 *        308, 128 x 128 378;  int8 6000 over 8, 2048 x 2048: 44, 128 x 128 53
    //             4096 of one, 4096 x 4096            118, 128 x 128 170;  16384 over 16, 1024 x 2048: 106, 128 x 128 108
    // Where the rule is not the faster side: 1024 over 64, 1024 x 1024 (16 rows an expert) rows 52, 64 x 64 tiles 42; 4096 over 8,
    // 2048 x 4096 128 x 128 116, 256 x 256 101.
    const long long groups = a.rows < a.experts ? a.rows : a.experts, avg = a.rows / a.experts;
    const auto tiles = [&](long long tm, long long tn) { return (a.rows / tm + groups) * ((a.n + tn - 1) / tn); };
    if (a.n <= 64 && a.k * z <= 256 && avg >= 512) {
        if (a.k * z <= 64) return a.n <= 32 ? run_narrow<T, 2, 1>(a, s) : run_narrow<T, 4, 1>(a, s);
        if (a.k * z <= 128) return a.n <= 32 ? run_narrow<T, 2, 2>(a, s) : run_narrow<T, 4, 2>(a, s);
        return a.n <= 32 ? run_narrow<T, 2, 4>(a, s) : run_narrow<T, 4, 4>(a, s);
    }
    if (tiles(32, 32) < 128) return run_rows<T, 1, 256, 8, 1, 160>(a, al, s);
    if (avg <= 24 && a.k * z <= 512) return run_rows<T, 1, 256, 1, 4, 40>(a, al, s);  // nothing to split k for: 61 rows over 82, 2334 x 71 int8: 14.8 us, split 35
    if (avg <= 4) return run_rows<T, 1, 128, 4, 2, 80>(a, al, s);
    if (tiles(64, 64) < (sizeof(T) == 4 ? 160 : 64)) return run_rows<T, 2, 128, 4, 2, 80>(a, al, s);
    if (avg <= 24) return run_rows<T, 4, 128, 2, 4, 80>(a, al, s);
    if (tiles(128, 128) < (sizeof(T) == 4 ? 1024 : 256)) return run_tile<T, 64, 64, 2, 2>(a, al, s);
    if constexpr (sizeof(T) < 4) {
        if (al && avg >= 256 && tiles(256, 256) >= (a.k >= 2048 ? 240 : 512)) return run_tile<T, 256, 256, 2, 4>(a, al, s);
    }
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
