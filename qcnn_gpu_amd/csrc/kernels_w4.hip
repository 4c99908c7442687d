// Products with 4-bit weights and group scales (qcnn_op_matvec_w4):
//   y[m][j] = sum_g s[g][j] sum_{k in g} (q[j][k] - z[g][j]) x[m][k] + b[j]
//
// Reading the weights is the cost, n * k / 2 bytes; everything else has to keep out of their way.  The codes become
// exact small numbers in the type of the matrix instruction (half or bfloat16), 16 x 16 x 32 tiles multiply them with up
// to 16 rows of x at a time, and the group's scale is applied to the float32 sums of the group, one multiplication for
// 32 to 128 weights.  One row of x costs as much as sixteen.
//
// The waves of a workgroup are KW x NW: NW share out the outputs, 16 NT each, KW the k, in runs of 128, and the KW sums
// meet in LDS at the end.  Everything goes through LDS, brought there by direct loads R - 1 runs ahead of its use, so that
// a wave has kilobytes on their way without registers for them (R is what LDS holds: 2 to 8; 2 for 5 to 16 rows and many outputs).  A wave issues an instruction every seven cycles or so, so
// instructions a run and waves on a CU set the pace where the memory does not.  A wave brings its own codes and scales; x is
// shared by the NW waves of a k group, one barrier a run, none for NW = 1.
// Measured, weights cold: 16 half rows, 16384 x 8192, groups of 64 with zeros: 27.5 us, 2.7 TB/s; one bfloat16 row, 4096 x 4096: 5.8 us.
// Of 128 k a lane holds 16 bytes of each of its weight rows: lane l, row l & 15, k from (l >> 4) * 32 on.  Instruction j
// of four wants k = 32 j + (l >> 4) * 8 there, so that its 32 k lie in one group: a 4 x 4 transposition of dwords among
// the lanes l, l + 16, l + 32, l + 48, four swaps of rows of lanes.
//
// Codes to numbers: 16 + q has q as the upper four bits of its fraction.  A byte b holds two codes; b * (1 + 2^12), shifted
// to the fraction by the same multiplication, has both in place, one in each half; and-or cuts them out and puts the
// exponents in: two operations for two weights, of which the multiplication picks the byte by itself.  The 16 and the
// zero point leave by the sum of x, a product of the same operand with ones:  sum (16 + q) x - (16 + z) sum x.  (Numbers of
// 16 to 31 where -8 to 7 are meant cost five times the rounding that -8 to 7 have: in the mean 1.0e-7 to 2.5e-7 of the L2 norm
// of an output's terms at k = 4096, where the library's float32 product has 5.7e-7.  Exact codes, -8 to 7 by v_cvt_off_f32_i4 or
// by half arithmetic, took 12 to 14 operations for 8 weights in place of 8 and the time was theirs.)
// float32 x: three bfloat16 parts (8 + 8 + 8 bits; exact down to 2^-109, below that multiples of 2^-133), three instructions.  Its
// results have the bits to show the rounding of larger sums and its time is that of the parts, so its codes are q - 8, and the
// sum of x comes in only with zero points.
#include "block_ops.h"

namespace qcnn {

#pragma clang diagnostic ignored "-Winline-asm"  // m0 in the clobber lists of the direct loads

// x as it is loaded (RAW registers of 4 for 8 values) and as the matrix instruction takes it (PARTS operands)
template <typename T>
struct XForm {
    static constexpr int RAW = 1, PARTS = 1;
};
template <>
struct XForm<float> {
    static constexpr int RAW = 2, PARTS = 3;
};

__device__ __forceinline__ unsigned upper_halves(unsigned lo, unsigned hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302); }

__device__ __forceinline__ void x_operand(f16_t, const u32x4 *raw, u32x4 *out) { out[0] = raw[0]; }
__device__ __forceinline__ void x_operand(bf16_t, const u32x4 *raw, u32x4 *out) { out[0] = raw[0]; }
__device__ __forceinline__ void x_operand(float, const u32x4 *raw, u32x4 *out)
{
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        unsigned a[2], b[2], c[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            a[i] = raw[p >> 1][(p & 1) * 2 + i];
            const float r = __uint_as_float(a[i]) - __uint_as_float(a[i] & 0xffff0000u);
            b[i] = __float_as_uint(r);
            c[i] = __float_as_uint(r - __uint_as_float(b[i] & 0xffff0000u));
        }
        out[0][p] = upper_halves(a[0], a[1]);
        out[1][p] = upper_halves(b[0], b[1]);
        out[2][p] = upper_halves(c[0], c[1]);
    }
}

// (byte B of v) * by
template <int B>
__device__ __forceinline__ unsigned byte_times(unsigned v, unsigned by)
{
    unsigned o;
    if constexpr (B == 0) asm("v_mul_u32_u24_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0 src1_sel:DWORD" : "=v"(o) : "v"(v), "v"(by));
    if constexpr (B == 1) asm("v_mul_u32_u24_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1 src1_sel:DWORD" : "=v"(o) : "v"(v), "v"(by));
    if constexpr (B == 2) asm("v_mul_u32_u24_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2 src1_sel:DWORD" : "=v"(o) : "v"(v), "v"(by));
    if constexpr (B == 3) asm("v_mul_u32_u24_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3 src1_sel:DWORD" : "=v"(o) : "v"(v), "v"(by));
    return o;
}
__device__ __forceinline__ unsigned and_or(unsigned v, unsigned mask, unsigned magic)
{
    unsigned o;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(o) : "v"(v), "s"(mask), "v"(magic));
    return o;
}

// (nibble 0 of byte B of v as two's complement) / 16, a float32 whose upper half is the bfloat16
template <int B>
__device__ __forceinline__ unsigned sixteenths(unsigned v)
{
    unsigned o;
    if constexpr (B == 0) asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(o) : "v"(v));
    if constexpr (B == 1) asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(o) : "v"(v));
    if constexpr (B == 2) asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(o) : "v"(v));
    if constexpr (B == 3) asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(o) : "v"(v));
    return o;
}

// The 8 codes of a dword as (q + ADD) / DIV, and the ones that go with them
template <typename T>
struct Codes {  // bfloat16
    static constexpr float ADD = 16.f, DIV = 1.f;
    static constexpr unsigned BY = 1 << 3 | 1 << 15, MASK = 0x00780078, MAGIC = 0x41804180, ONES = 0x3f803f80;
};
template <>
struct Codes<f16_t> {
    static constexpr float ADD = 16.f, DIV = 1.f;
    static constexpr unsigned BY = 1 << 6 | 1 << 18, MASK = 0x03c003c0, MAGIC = 0x4c004c00, ONES = 0x3c003c00;
};
template <>
struct Codes<float> {
    static constexpr float ADD = -8.f, DIV = 16.f;
    static constexpr unsigned ONES = 0x3f803f80;
};
template <typename T>
__device__ __forceinline__ u32x4 codes(unsigned w)
{
    typedef Codes<T> C;
    if constexpr (__is_same(T, float)) {
        const unsigned even = w ^ 0x88888888u, odd = even >> 4;  // two's complement of q - 8
        return u32x4{upper_halves(sixteenths<0>(even), sixteenths<0>(odd)), upper_halves(sixteenths<1>(even), sixteenths<1>(odd)),
                     upper_halves(sixteenths<2>(even), sixteenths<2>(odd)), upper_halves(sixteenths<3>(even), sixteenths<3>(odd))};
    } else
    return u32x4{and_or(byte_times<0>(w, C::BY), C::MASK, C::MAGIC), and_or(byte_times<1>(w, C::BY), C::MASK, C::MAGIC),
                 and_or(byte_times<2>(w, C::BY), C::MASK, C::MAGIC), and_or(byte_times<3>(w, C::BY), C::MASK, C::MAGIC)};
}

__device__ __forceinline__ f32x4 mma(float, u32x4 x, u32x4 w, f32x4 c) { return mma(bf16_t(), x, w, c); }

// dwords j of lanes l, l + 16, l + 32, l + 48 change places: lane l + 16 i's dword j goes to lane l + 16 j's dword i
__device__ __forceinline__ u32x4 transpose4(u32x4 v)
{
    // rows of 16 lanes 0 1 2 3: first the halves (0 1 | 2 3) of dwords 0, 2 and 1, 3, then neighbours of dwords 0, 1 and 2, 3
    u32x2 a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false), b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
    u32x2 c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return u32x4{c[0], c[1], d[0], d[1]};
}

// Direct loads to LDS from a uniform address and the lane's offset: lane l's 16 bytes go to lds + 16 l, or its one
// element of N bytes to lds + 4 l.  (The s_nop holds the wait states that the load
// needs behind the write of m0, one, and behind a vector instruction's write of the address registers, five.)
__device__ __forceinline__ void lds_load16(unsigned lds, unsigned offset, const char *base)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void lds_load_one(unsigned lds, unsigned offset, const char *base)
{
    if constexpr (N == 1)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_ubyte %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory", "m0");
    else if constexpr (N == 2)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_ushort %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ const char *uniform(const char *p)
{
    const unsigned long long u = (unsigned long long)p;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)u), hi = __builtin_amdgcn_readfirstlane((unsigned)(u >> 32));  // (it returns int)
    return (const char *)((unsigned long long)hi << 32 | lo);
}

// LDS of one run of 128 k: x of XROWS rows for the NW waves, then for each wave its codes (1 KB a tile of 16 outputs) and
// the scales and zero points of its outputs, a dword each, one set for FL instructions.  Chunk c of 16 bytes of x row r stands in slot c ^ (r & 15) of
// its row: the sixteen lanes that a ds_read_b128 serves at a time read different slots of the 256 bytes that the banks hold.
template <typename T, int NT, int XROWS, int FL, bool S16, bool ZERO, int KW, int NW, int KB>
struct W4 {
    static constexpr int WAVES = KW * NW, MT = XROWS < 16 ? 1 : XROWS / 16;
    static constexpr int XB = XROWS * 128 * (int)sizeof(T), NS = 4 / FL, SB = NS * NT * 64, SI = (SB + 255) / 256;
    static constexpr int WB = NT * 1024 + SI * 256 * (ZERO ? 2 : 1), RUN = XB + NW * WB;
    static constexpr int LOADS = NT + XB / 1024 / NW + SI * (ZERO ? 2 : 1);  // direct loads of a wave for one run
    static constexpr int FIT = KB * 1024 / (KW * RUN), R = FIT < 2 ? 2 : FIT < 8 ? FIT : 8;  // runs in the ring: as many as KB kilobytes hold
    static constexpr int SUMS = WAVES * NT * MT * 1024;
    static constexpr int LDS = KW * R * RUN > SUMS ? KW * R * RUN : SUMS;
    static_assert(XB / 1024 % NW == 0 && NT <= 4 && LOADS * (R - 2) < 64 && LDS <= 163840, "runs fit");
};

// S16: scales of 16 bits; ZERO: zero points are given.
template <typename T, int NT, int XROWS, int FL, bool S16, bool ZERO, int KW, int NW, int KB>
__global__ __launch_bounds__(64 * KW *NW) void k_w4(const qcnn_matvec_w4_t a, unsigned nblocks)
{
    typedef W4<T, NT, XROWS, FL, S16, ZERO, KW, NW, KB> G;
    constexpr int PARTS = XForm<T>::PARTS, RAW = XForm<T>::RAW, MT = G::MT, NS = G::NS, R = G::R, TS = sizeof(T), SS = S16 ? 2 : 4;
    extern __shared__ __align__(1024) char lds[];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c16 = lane & 15, g = lane >> 4;
    const int kq = wave / NW, nq = wave % NW;
    const int n0 = ((int)(blockIdx.x % nblocks) * NW + nq) * 16 * NT, m0 = (int)(blockIdx.x / nblocks) * XROWS;
    const int rows = min(XROWS, a.rows - m0), row_bytes = (a.k + 1) >> 1;

    // runs of this k group: pairs, as two runs share the cache lines of the weight rows; the last run of all may be cut by
    // the end of the rows.  Every wave of the workgroup makes `turns` turns.
    const int all = (a.k + 127) >> 7, turns = ((all + 1) / 2 + KW - 1) / KW * 2;
    const int first = kq * turns, count = max(0, min(turns, all - first));
    const bool cut = a.k % 128 != 0 && first + count == all && count > 0;
    const int whole = count - (cut ? 1 : 0);

    // this lane's sources, as offsets from uniform addresses (ldw and ldx are at most 2^25 and 2^24)
    unsigned wat[NT], xat[G::XB / 1024 / NW];
#pragma unroll
    for (int t = 0; t < NT; ++t) wat[t] = (unsigned)max(0, min(t * 16 + c16, a.n - 1 - n0)) * (unsigned)a.ldw + g * 16;
    constexpr int CPR = 8 * TS;  // chunks of an x row
#pragma unroll
    for (int i = 0; i < G::XB / 1024 / NW; ++i) {
        const int at = (i * NW + nq) * 64 + lane, row = at / CPR;
        xat[i] = (unsigned)min(row, rows - 1) * (unsigned)(a.ldx * TS) + ((at % CPR) ^ (row & 15)) * 16;
    }
    const int nbase = min(n0, a.n - 1);  // (a wave beyond the outputs reads the last one's and stores nothing)
    const unsigned per = (unsigned)a.group >> 5;  // 32s of k in a group
    char *const ring = lds + kq * (R * G::RUN);
    const unsigned ring_at = (unsigned)(size_t)(__attribute__((address_space(3))) char *)ring;

    // What moves from run to run, in scalar registers: a wave has few companions to hide a long scalar sum behind.
    const char *w = uniform((const char *)a.w + (size_t)nbase * a.ldw + (size_t)first * 64);
    const char *x = uniform((const char *)a.x + ((size_t)m0 * a.ldx + (size_t)first * 128) * TS);
    const unsigned group = (unsigned)first * 4 / per;
    unsigned used = (unsigned)first * 4 % per;  // 32s of k of the next run's group that are behind us
    const char *sc = uniform((const char *)a.scale + ((size_t)group * a.n + nbase) * SS);
    const char *zp = uniform((const char *)a.zero + (size_t)group * a.n + nbase);
    int bring_slot = 0;
    // Scale e = 64 i + lane of a run is that of set e / 16 NT, output e % 16 NT.  With groups of 32, 64 or whole 128s the sets of
    // every run lie at the same distances (n <= 2^26: they fit).
    const bool steady = FL == 4 || per <= 2;
    unsigned col[G::SI], offset[G::SI];
    int set[G::SI];
#pragma unroll
    for (int i = 0; i < G::SI; ++i) {
        set[i] = min((i * 64 + lane) / (16 * NT), NS - 1);
        col[i] = (unsigned)max(0, min((i * 64 + lane) % (16 * NT), a.n - 1 - n0));
        offset[i] = col[i] + (FL == 4 ? 0u : (unsigned)(set[i] * FL) / per * (unsigned)a.n);
    }
    const auto sets_of_run = [&] {  // offset[] where they do not
        unsigned step[NS], u = used, d = 0;
#pragma unroll
        for (int f = 0; f < NS; ++f) {
            step[f] = d;
            u += FL;
            if (u == per) u = 0, ++d;
        }
#pragma unroll
        for (int i = 0; i < G::SI; ++i) {
            unsigned by = 0;
#pragma unroll
            for (int f = 1; f < NS; ++f)
                if (set[i] == f) by = step[f];
            offset[i] = col[i] + by * (unsigned)a.n;
        }
    };
    // brings run i (of this group) into the ring; called for 0, 1, 2 ...
    const auto bring = [&](int i) {
        if (i < whole) {
            const unsigned at = ring_at + bring_slot, mine = at + G::XB + nq * G::WB;
#pragma unroll
            for (int t = 0; t < NT; ++t) lds_load16(mine + t * 1024, wat[t], w);
#pragma unroll
            for (int j = 0; j < G::XB / 1024 / NW; ++j) lds_load16(at + (j * NW + nq) * 1024, xat[j], x);
            if (!steady) sets_of_run();
#pragma unroll
            for (int j = 0; j < G::SI; ++j) {
                lds_load_one<SS>(mine + NT * 1024 + j * 256, offset[j] * SS, sc);
                if (ZERO) lds_load_one<1>(mine + NT * 1024 + (G::SI + j) * 256, offset[j], zp);
            }
            w += 64;
            x += 128 * TS;
            used += 4;
            while (used >= per) {  // (at most four times)
                used -= per;
                sc += (size_t)a.n * SS;
                zp += a.n;
            }
        } else if (cut && i == whole) {  // element by element, zeros behind the end of x
            const int kb = first + i;
            char *at = ring + bring_slot, *mine = at + G::XB + nq * G::WB;
            // (eight loads on their way at a time: one at a time cost 5 x 1001 x 2047 float32 1.8 us more)
#pragma unroll 1
            for (int t = 0; t < 2 * NT; ++t) {  // of 8 rows the lane brings byte lane; lane (row + 16 (byte >> 4)) of their tile reads it
                uint8_t v[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) v[r] = kb * 64 + lane < row_bytes && n0 + t * 8 + r < a.n ? w[(size_t)(t * 8 + r) * a.ldw + lane] : 0;
#pragma unroll
                for (int r = 0; r < 8; ++r) mine[(t >> 1) * 1024 + ((lane >> 4) * 16 + (t & 1) * 8 + r) * 16 + (lane & 15)] = v[r];
            }
            constexpr int EACH = XROWS * 128 / (NW * 64), BATCH = EACH < 8 ? EACH : 8;
            static_assert(XROWS * 128 % (NW * 64) == 0 && EACH % BATCH == 0, "whole batches");
#pragma unroll 1
            for (int e0 = 0; e0 < EACH; e0 += BATCH) {
                T v[BATCH];
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const int e = ((e0 + i) * NW + nq) * 64 + lane, row = e >> 7, k = e & 127;
                    from_f32(0.f, v[i]);
                    if (kb * 128 + k < a.k) v[i] = ((const T *)x)[(size_t)min(row, rows - 1) * a.ldx + k];
                }
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const int e = ((e0 + i) * NW + nq) * 64 + lane, row = e >> 7, k = e & 127, c = k * TS / 16;
                    *(T *)(at + row * (128 * TS) + (c ^ (row & 15)) * 16 + k * TS % 16) = v[i];
                }
            }
            const unsigned last = (unsigned)(a.k - 1) / (unsigned)a.group;
#pragma unroll
            for (int j = 0; j < G::SI; ++j) {
                const size_t e = (size_t)min(((unsigned)kb * 4 + set[j] * FL) / per, last) * a.n + nbase + col[j];
                unsigned *sz = (unsigned *)(mine + NT * 1024 + j * 256) + lane;
                *sz = S16 ? ((const uint16_t *)a.scale)[e] : ((const unsigned *)a.scale)[e];
                if (kb * 128 + set[j] * (FL * 32) >= a.k) *sz = 0;  // behind the row's end x is zero: an infinite scale must not meet it
                if (ZERO) sz[G::SI * 64] = ((const uint8_t *)a.zero)[e];
            }
        }
        bring_slot = bring_slot == (R - 1) * G::RUN ? 0 : bring_slot + G::RUN;
    };

    f32x4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[t][m] = f32x4{0, 0, 0, 0};
    constexpr bool SUM_X = Codes<T>::ADD + 8.f != 0.f || ZERO;
    const bool bf16_scales = a.scale_type == QCNN_BF16;

    // a run in registers: everything is asked of LDS before the first of it is used
    struct Run {
        u32x4 w[NT], x[4][MT][RAW];
        unsigned s[NS][NT], z[NS][NT];
    };
    int slot = 0;
    const auto fetch = [&](Run &r) {
        const char *at = ring + slot, *mine = at + G::XB + nq * G::WB;
#pragma unroll
        for (int t = 0; t < NT; ++t) r.w[t] = *(const u32x4 *)(mine + t * 1024 + lane * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const int row = XROWS < 16 ? c16 % XROWS : m * 16 + c16;
#pragma unroll
                for (int i = 0; i < RAW; ++i) r.x[j][m][i] = *(const u32x4 *)(at + row * (128 * TS) + (((j * 4 + g) * RAW + i) ^ (row & 15)) * 16);
            }
#pragma unroll
        for (int f = 0; f < NS; ++f)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const char *p = mine + NT * 1024 + (f * 16 * NT + t * 16 + c16) * 4;
                r.s[f][t] = S16 ? *(const uint16_t *)p : *(const unsigned *)p;
                if (ZERO) r.z[f][t] = *(const uint8_t *)(p + G::SI * 256);
            }
        slot = slot == (R - 1) * G::RUN ? 0 : slot + G::RUN;
    };
    const auto compute = [&](const Run &r) {
        u32x4 w[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) w[t] = transpose4(r.w[t]);
#pragma unroll
        for (int f = 0; f < NS; ++f) {
            f32x4 sum[NT][MT], ones[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                ones[m] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < NT; ++t) sum[t][m] = f32x4{0, 0, 0, 0};
            }
#pragma unroll
            for (int j = f * FL; j < (f + 1) * FL; ++j) {
                u32x4 x[MT][PARTS];
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    x_operand(T(), r.x[j][m], x[m]);
                    if (SUM_X) {
                        const u32x4 one = {Codes<T>::ONES, Codes<T>::ONES, Codes<T>::ONES, Codes<T>::ONES};
#pragma unroll
                        for (int p = 0; p < PARTS; ++p) ones[m] = mma(T(), x[m][p], one, ones[m]);
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const u32x4 c = codes<T>(w[t][j]);
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int p = 0; p < PARTS; ++p) sum[t][m] = mma(T(), x[m][p], c, sum[t][m]);
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const unsigned u = r.s[f][t];
                const float s = !S16 ? __uint_as_float(u) : bf16_scales ? __uint_as_float(u << 16) : (float)__builtin_bit_cast(f16_t, (uint16_t)u);
                const float z = Codes<T>::ADD + (ZERO ? (float)r.z[f][t] : 8.f);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float v = Codes<T>::DIV * sum[t][m][q];
                        acc[t][m][q] = fmaf(s, SUM_X ? fmaf(-z, ones[m][q], v) : v, acc[t][m][q]);
                    }
            }
        }
    };

#pragma unroll 1
    for (int i = 0; i < R - 1; ++i) bring(i);
    for (int i = 0; i < turns; ++i) {
        // run i has landed (loads land in order: all but those of the runs behind it), here and after the barrier for all, and
        // everyone is done with run i - 1, whose place run i + R - 1 takes
        wait_for_all_but<R - 2, G::LOADS>(whole - 1 - i);
        if (NW > 1) asm volatile("s_barrier" ::: "memory");
        bring(i + R - 1);
        if (i < count) {
            Run r;
            fetch(r);
            compute(r);
        }
    }

    // the k groups' sums; the lane has rows 4 g .. 4 g + 3 of output c16 of each tile
    __syncthreads();
    float *sums = (float *)lds;
    constexpr int OUT = 16 * NT * NW;  // outputs of the workgroup
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int q = 0; q < 4; ++q) sums[kq * (OUT * 16 * MT) + (m * 16 + 4 * g + q) * OUT + nq * (16 * NT) + t * 16 + c16] = acc[t][m][q];
    __syncthreads();
    const int base = (int)(blockIdx.x % nblocks) * OUT;
    for (int o = threadIdx.x; o < OUT * rows; o += 64 * KW * NW) {
        const int row = o / OUT, j = base + o % OUT;
        if (j >= a.n) continue;
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < KW; ++k) v += sums[k * (OUT * 16 * MT) + o];
        if (a.bias) v += ((const float *)a.bias)[j];
        store_typed(a.y, (size_t)(m0 + row) * a.ldy + j, a.out_type, v);
    }
}

template <typename T, int NT, int XROWS, int FL, bool S16, bool ZERO, int KW, int NW, int KB>
static hipError_t launch(const qcnn_matvec_w4_t &a, hipStream_t s)
{
    typedef W4<T, NT, XROWS, FL, S16, ZERO, KW, NW, KB> G;
    const unsigned nblocks = (unsigned)((a.n + 16 * NT * NW - 1) / (16 * NT * NW));
    const auto fn = k_w4<T, NT, XROWS, FL, S16, ZERO, KW, NW, KB>;
    static std::atomic<unsigned long long> asked{0};
    const hipError_t e = allow_lds((const void *)fn, G::LDS, asked);
    if (e != hipSuccess) return e;
    // a launch's threads have to stay below 2^32: more rows take several (n <= 2^26: at least XROWS rows fit)
    const unsigned most = 0xffffffffu / (64 * G::WAVES) / nblocks;
    if (!most) return hipErrorNotSupported;
    qcnn_matvec_w4_t part = a;
    for (long long done = 0; done < a.rows; done += (long long)most * XROWS) {
        part.rows = (int)(a.rows - done < (long long)most * XROWS ? a.rows - done : (long long)most * XROWS);
        part.x = (const char *)a.x + (size_t)done * a.ldx * sizeof(T);
        part.y = (char *)a.y + (size_t)done * a.ldy * (a.out_type == QCNN_F32 ? 4 : 2);
        fn<<<nblocks * (((unsigned)part.rows + XROWS - 1) / XROWS), 64 * G::WAVES, G::LDS, s>>>(part, nblocks);
        const hipError_t launched = hipGetLastError();
        if (launched != hipSuccess) return launched;
    }
    return hipSuccess;
}

template <typename T, int NT, int XROWS, int FL, int KW, int NW, int KB>
static hipError_t run(const qcnn_matvec_w4_t &a, hipStream_t s)
{
    if (a.scale_type != QCNN_F32)
        return a.zero ? launch<T, NT, XROWS, FL, true, true, KW, NW, KB>(a, s) : launch<T, NT, XROWS, FL, true, false, KW, NW, KB>(a, s);
    return a.zero ? launch<T, NT, XROWS, FL, false, true, KW, NW, KB>(a, s) : launch<T, NT, XROWS, FL, false, false, KW, NW, KB>(a, s);
}

// Rows of x a workgroup takes and how its waves share out the work.  With few outputs there are few workgroups, each
// wave is alone with its instructions' latencies, and more waves along k are what helps; with many outputs, sharing x
// among waves and several workgroups on a CU.  Microseconds at k = 4096, group 128, for n = 1024 / 4096 / 8192 / 16384 (a call of a
// captured graph of calls, median of 9, weights cold), the taken side of each border first:
//   bfloat16 rows <= 4     4.7 / 5.8 / 7.6 / 11.5   (KB 80: 4.7 / 6.0 / 8.0 / 13.2;  two tiles a wave 6.1 / 7.0 / 7.5 / 11.2)
//            rows <= 16    8 x 1 5.4 / 6.9 / 11.8 / 22 up to 4096, 4 x 2 7.5 / 8.3 / 8.8 / 13.9 above
//            32 rows       4 x 2 9.3 / 10.8 / 11.4 / 21.2 up to 4096, 4 x 4 12.4 / 14.1 / 14.3 / 16.6 above
//            64 rows       32 rows 4 x 2 9.4 / 11.0 / 20.0 / 38 up to 4096, 4 x 4 12.4 / 13.8 / 15.3 / 28.4 up to 8192, 64 rows 2 x 4
//                          20.8 / 22.6 / 22.8 / 25.0 above
//   float32  rows <= 4     one tile 7.4 / 8.0 / 12.0 / 21.0 up to 4096, two 8.8 / 9.4 / 9.9 / 16.3 above
//            rows <= 16    one tile 12.8 / 14.1 / 14.6 / 27.1 up to 8192, two 17.6 / 19.3 / 19.7 / 21.1 above
//            64 rows       16 rows 4 x 4 20.2 / 21.2 / 40.2 / 79 up to 8192 (and up to 32 rows), 32 rows, two tiles 45 / 47 / 48 / 49.4
//                          above
// (Not the faster side: bfloat16 32 rows at n = 8192 4 x 2 11.4; float32 16 rows at n = 4096 8 x 1 9.8.)
// Where that leaves fewer than 128 workgroups, sixteen rows and sixteen outputs each with the most waves along k that fit:
// 9 x 167 x 12134 float32 46 -> 21 us, 22 x 128 x 10048 bfloat16 22 -> 11.6.
template <typename T, int FL>
static hipError_t pick_rows(const qcnn_matvec_w4_t &a, hipStream_t s)
{
    constexpr bool F = sizeof(T) == 4;
    const auto groups = [&](long long rows, long long outputs) { return ((a.rows + rows - 1) / rows) * ((a.n + outputs - 1) / outputs); };
    if (a.rows <= 4) {
        if (groups(4, 16) < 128) return run<T, 1, 4, FL, 16, 1, F ? 160 : 106>(a, s);
        if constexpr (F) return a.n <= 4096 ? run<T, 1, 4, FL, 8, 1, 80>(a, s) : run<T, 2, 4, FL, 8, 1, 80>(a, s);
        return run<T, 1, 4, FL, 8, 1, 53>(a, s);
    }
    if (groups(32, 32) < 128) return run<T, 1, 16, FL, 8, 1, 160>(a, s);
    if constexpr (F) {
        if (a.rows <= 16) return a.n <= 8192 ? run<T, 1, 16, FL, 4, 2, 80>(a, s) : run<T, 2, 16, FL, 4, 2, 160>(a, s);
        return a.rows <= 32 || a.n <= 8192 ? run<T, 1, 16, FL, 4, 4, 160>(a, s) : run<T, 2, 32, FL, 2, 4, 160>(a, s);
    } else {
        if (a.rows <= 16) return a.n <= 4096 ? run<T, 1, 16, FL, 8, 1, 160>(a, s) : run<T, 1, 16, FL, 4, 2, 80>(a, s);
        if (a.n <= 4096) return run<T, 1, 32, FL, 4, 2, 160>(a, s);
        return a.rows <= 32 || a.n <= 8192 ? run<T, 1, 32, FL, 4, 4, 160>(a, s) : run<T, 1, 64, FL, 2, 4, 160>(a, s);
    }
}

template <typename T>
static hipError_t pick(const qcnn_matvec_w4_t &a, hipStream_t s)
{
    if (a.group % 128 == 0) return pick_rows<T, 4>(a, s);
    if (a.group % 64 == 0) return pick_rows<T, 2>(a, s);
    return pick_rows<T, 1>(a, s);
}

hipError_t launch_matvec_w4(const qcnn_matvec_w4_t &a, hipStream_t s)
{
    if (a.type == QCNN_F32) return pick<float>(a, s);
    if (a.type == QCNN_F16) return pick<f16_t>(a, s);
    return pick<bf16_t>(a, s);
}

}  // namespace qcnn
