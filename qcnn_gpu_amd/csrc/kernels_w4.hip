// Products with 4-bit weights and group scales (qcnn_op_matvec_w4):
//   y[m][j] = sum_g s[g][j] sum_{k in g} (q[j][k] - z[g][j]) x[m][k] + b[j]
//
// Reading the weights is the cost, n * k / 2 bytes; everything else has to keep out of their way.  The codes become
// exact small integers in the type of the matrix instruction (half or bfloat16), 16 x 16 x 32 tiles multiply them with up
// to 16 rows of x at a time, and the group's scale is applied to the float32 sums of the group, one multiplication for
// 32 to 128 weights.  One row of x costs as much as sixteen.
//
// The waves of a workgroup are KW x NW: NW share out the outputs, 16 NT each, KW the k, in runs of 128, and the KW sums
// meet in LDS at the end.  Everything goes through LDS, brought there by direct loads R - 1 runs ahead of its use, so that
// a wave has kilobytes on their way without registers for them (with loads into registers the compiler's waits left
// little in flight: 2.8 TB/s).  A wave brings its own codes and scales; x is shared by the NW waves of a k group, one
// barrier a run, none for NW = 1.
// Of 128 k a lane holds 16 bytes of each of its weight rows: lane l, row l & 15, k from (l >> 4) * 32 on.  Instruction j
// of four wants k = 32 j + (l >> 4) * 8 there, so that its 32 k lie in one group: a 4 x 4 transposition of dwords among
// the lanes l, l + 16, l + 32, l + 48, four swaps of rows of lanes.
//
// Codes to half: (w & 0x000f000f) | 0x64006400 is the pair 1024 + q of the nibbles 0 and 4, minus (1024 + z) exact; nibbles
// 1 and 5 from 0x00f000f0 as 1024 + 16 q, times 1/16 minus (64 + z); the other four the same from w >> 8: 9 operations for
// 8 weights.  x comes in the same order of pairs, four v_perm_b32 for 8 values.
// Codes to bfloat16: v_cvt_off_f32_i4 makes (q - 8) / 16 of a nibble, whose upper half is the bfloat16: 14 operations for
// 8 weights.  Zero points other than 8 come in by sums of x (a product with ones): s (8 - z) sum x.
// float32 x: three bfloat16 parts (8 + 8 + 8 bits, exact), three instructions.
#include "block_ops.h"

namespace qcnn {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef u32x4 u32x4_any __attribute__((aligned(1)));

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

__device__ __forceinline__ u32x4 perm4(u32x4 v)  // elements (0,4) (1,5) (2,6) (3,7)
{
    return u32x4{__builtin_amdgcn_perm(v[2], v[0], 0x05040100), __builtin_amdgcn_perm(v[2], v[0], 0x07060302),
                 __builtin_amdgcn_perm(v[3], v[1], 0x05040100), __builtin_amdgcn_perm(v[3], v[1], 0x07060302)};
}
__device__ __forceinline__ unsigned upper_halves(unsigned lo, unsigned hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302); }

__device__ __forceinline__ void x_operand(f16_t, const u32x4 *raw, u32x4 *out) { out[0] = perm4(raw[0]); }
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

// (v & mask) | magic and the conversion of nibble 0 of byte B, one instruction each (the compiler makes two of both)
__device__ __forceinline__ unsigned and_or(unsigned v, unsigned mask, unsigned magic)
{
    unsigned o;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(o) : "v"(v), "s"(mask), "v"(magic));
    return o;
}
template <int B>
__device__ __forceinline__ unsigned sixteenths(unsigned v)
{
    unsigned o;
    if constexpr (B == 0) asm("v_cvt_off_f32_i4_e32 %0, %1" : "=v"(o) : "v"(v));
    if constexpr (B == 1) asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(o) : "v"(v));
    if constexpr (B == 2) asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(o) : "v"(v));
    if constexpr (B == 3) asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(o) : "v"(v));
    return o;
}

// 8 codes of a dword as the other operand; z: the pair of constants of a half operand (unused otherwise)
struct HalfZero {
    f16x2 low, high;  // -(1024 + z), -(64 + z)
};
__device__ __forceinline__ HalfZero half_zero(float z)
{
    const f16_t a = (f16_t)(-1024.f - z), b = (f16_t)(-64.f - z);
    return HalfZero{f16x2{a, a}, f16x2{b, b}};
}
__device__ __forceinline__ u32x4 codes(f16_t, unsigned w, const HalfZero &z)
{
    const f16x2 r = {(f16_t)0.0625f, (f16_t)0.0625f};
    u32x4 o;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const unsigned v = h ? w >> 8 : w;
        const f16x2 a = __builtin_bit_cast(f16x2, and_or(v, 0x000f000fu, 0x64006400u)), b = __builtin_bit_cast(f16x2, and_or(v, 0x00f000f0u, 0x64006400u));
        o[2 * h] = __builtin_bit_cast(unsigned, (f16x2)(a + z.low));
        o[2 * h + 1] = __builtin_bit_cast(unsigned, __builtin_elementwise_fma(b, r, z.high));
    }
    return o;
}
__device__ __forceinline__ u32x4 codes(bf16_t, unsigned w, const HalfZero &)
{
    const unsigned even = w ^ 0x88888888u, odd = even >> 4;  // two's complement of q - 8
    return u32x4{upper_halves(sixteenths<0>(even), sixteenths<0>(odd)), upper_halves(sixteenths<1>(even), sixteenths<1>(odd)),
                 upper_halves(sixteenths<2>(even), sixteenths<2>(odd)), upper_halves(sixteenths<3>(even), sixteenths<3>(odd))};
}
__device__ __forceinline__ u32x4 codes(float, unsigned w, const HalfZero &z) { return codes(bf16_t(), w, z); }

__device__ __forceinline__ f32x4 mma(f16_t, u32x4 x, u32x4 w, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, w), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(bf16_t, u32x4 x, u32x4 w, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, w), c, 0, 0, 0);
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
template <typename T, int NT, int XROWS, int FL, bool S16, bool ZERO, int KW, int NW, int R>
struct W4 {
    static constexpr int WAVES = KW * NW, MT = XROWS < 16 ? 1 : XROWS / 16;
    static constexpr int XB = XROWS * 128 * (int)sizeof(T), NS = 4 / FL, SB = NS * NT * 64, SI = (SB + 255) / 256;
    static constexpr int WB = NT * 1024 + SI * 256 * (ZERO ? 2 : 1), RUN = XB + NW * WB;
    static constexpr int LOADS = NT + XB / 1024 / NW + SI * (ZERO ? 2 : 1);  // direct loads of a wave for one run
    static constexpr int SUMS = WAVES * NT * MT * 1024;
    static constexpr int LDS = KW * R * RUN > SUMS ? KW * R * RUN : SUMS;
    static_assert(XB / 1024 % NW == 0 && NT <= 4 && LOADS * (R - 2) < 64 && LDS <= 163840, "runs fit");
};

// S16: scales of 16 bits; ZERO: zero points are given.
template <typename T, int NT, int XROWS, int FL, bool S16, bool ZERO, int KW, int NW, int R>
__global__ __launch_bounds__(64 * KW *NW) void k_w4(const qcnn_matvec_w4_t a, unsigned nblocks)
{
    typedef W4<T, NT, XROWS, FL, S16, ZERO, KW, NW, R> G;
    constexpr int PARTS = XForm<T>::PARTS, RAW = XForm<T>::RAW, MT = G::MT, NS = G::NS, TS = sizeof(T), SS = S16 ? 2 : 4;
    constexpr bool HALF = __is_same(T, f16_t);
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
    // scale e = 64 i + lane of a run: of set e / 16 NT, output e % 16 NT
    unsigned col[G::SI];
    int set[G::SI];
#pragma unroll
    for (int i = 0; i < G::SI; ++i) {
        set[i] = min((i * 64 + lane) / (16 * NT), NS - 1);
        col[i] = (unsigned)max(0, min((i * 64 + lane) % (16 * NT), a.n - 1 - n0));
    }
    const int nbase = min(n0, a.n - 1);  // (a wave beyond the outputs reads the last one's and stores nothing)
    const char *const w0 = (const char *)a.w + (size_t)nbase * a.ldw, *const x0 = (const char *)a.x + (size_t)m0 * a.ldx * TS;
    const unsigned per = (unsigned)a.group >> 5, last = (unsigned)(a.k - 1) / (unsigned)a.group;
    char *const ring = lds + kq * (R * G::RUN);
    const unsigned ring_at = (unsigned)(size_t)(__attribute__((address_space(3))) char *)ring;

    unsigned gi = (unsigned)first * 4 / per, left = per - (unsigned)first * 4 % per;  // group of the next run to bring, its 32s of k left
    const auto next_scales = [&](size_t &from, unsigned (&offset)[G::SI]) {  // elements: of the first set, and of each lane's from there
        unsigned group[NS];
#pragma unroll
        for (int f = 0; f < NS; ++f) {
            group[f] = min(gi, last);  // (behind the last group x is zero)
            left -= FL;
            if (left == 0) ++gi, left = per;
        }
        from = (size_t)group[0] * a.n + nbase;
#pragma unroll
        for (int i = 0; i < G::SI; ++i) {
            offset[i] = col[i];
#pragma unroll
            for (int f = 1; f < NS; ++f)
                if (set[i] == f) offset[i] += (group[f] - group[0]) * (unsigned)a.n;  // (n <= 2^26)
        }
    };
    // brings run i (of this group) into the ring
    const auto bring = [&](int i) {
        const int kb = first + i, slot = i % R;
        if (i < whole) {
            const unsigned at = ring_at + slot * G::RUN, mine = at + G::XB + nq * G::WB;
            const char *w = uniform(w0 + (size_t)kb * 64), *x = uniform(x0 + (size_t)kb * (128 * TS));
#pragma unroll
            for (int t = 0; t < NT; ++t) lds_load16(mine + t * 1024, wat[t], w);
#pragma unroll
            for (int j = 0; j < G::XB / 1024 / NW; ++j) lds_load16(at + (j * NW + nq) * 1024, xat[j], x);
            size_t from;
            unsigned offset[G::SI];
            next_scales(from, offset);
#pragma unroll
            for (int j = 0; j < G::SI; ++j) {
                lds_load_one<SS>(mine + NT * 1024 + j * 256, offset[j] * SS, uniform((const char *)a.scale + from * SS));
                if (ZERO) lds_load_one<1>(mine + NT * 1024 + (G::SI + j) * 256, offset[j], uniform((const char *)a.zero + from));
            }
        } else if (cut && i == whole) {  // element by element, zeros behind the end of x
            char *at = ring + slot * G::RUN, *mine = at + G::XB + nq * G::WB;
            for (int e = lane; e < NT * 1024; e += 64) {  // byte e & 63 of weight row e >> 6; lane (row & 15) + 16 (byte >> 4) reads it
                const int row = e >> 6, byte = e & 63;
                mine[(row >> 4) * 1024 + ((byte >> 4) * 16 + (row & 15)) * 16 + (byte & 15)] =
                    kb * 64 + byte < row_bytes && n0 + row < a.n ? w0[(size_t)row * a.ldw + kb * 64 + byte] : 0;
            }
            T zero;
            from_f32(0.f, zero);
            for (int e = nq * 64 + lane; e < XROWS * 128; e += NW * 64) {
                const int row = e >> 7, k = e & 127, c = k * TS / 16;
                *(T *)(at + row * (128 * TS) + (c ^ (row & 15)) * 16 + k * TS % 16) =
                    kb * 128 + k < a.k ? ((const T *)x0)[(size_t)min(row, rows - 1) * a.ldx + kb * 128 + k] : zero;
            }
            size_t from;
            unsigned offset[G::SI];
            next_scales(from, offset);
#pragma unroll
            for (int j = 0; j < G::SI; ++j) {
                unsigned *sz = (unsigned *)(mine + NT * 1024 + j * 256) + lane;
                *sz = S16 ? ((const uint16_t *)a.scale)[from + offset[j]] : ((const unsigned *)a.scale)[from + offset[j]];
                if (ZERO) sz[G::SI * 64] = ((const uint8_t *)a.zero)[from + offset[j]];
            }
        }
    };

    f32x4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[t][m] = f32x4{0, 0, 0, 0};
    const bool bf16_scales = a.scale_type == QCNN_BF16;

    const auto consume = [&](int i) {
        const char *at = ring + i % R * G::RUN, *mine = at + G::XB + nq * G::WB;
        u32x4 w[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) w[t] = transpose4(*(const u32x4 *)(mine + t * 1024 + lane * 16));
#pragma unroll
        for (int f = 0; f < NS; ++f) {
            f32x4 sum[NT][MT], ones[MT];
            float s[NT], z[NT];
            HalfZero hz[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const char *p = mine + NT * 1024 + (f * 16 * NT + t * 16 + c16) * 4;
                if (S16) {
                    const unsigned u = *(const uint16_t *)p;
                    s[t] = bf16_scales ? __uint_as_float(u << 16) : (float)__builtin_bit_cast(f16_t, (uint16_t)u);
                } else {
                    s[t] = *(const float *)p;
                }
                z[t] = ZERO ? (float)*(const uint8_t *)(p + G::SI * 256) : 8.f;
                hz[t] = half_zero(z[t]);
            }
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
                    const int row = XROWS < 16 ? c16 % XROWS : m * 16 + c16;
                    u32x4 raw[RAW];
#pragma unroll
                    for (int r = 0; r < RAW; ++r)
                        raw[r] = *(const u32x4 *)(at + row * (128 * TS) + (((j * 4 + g) * RAW + r) ^ (row & 15)) * 16);
                    x_operand(T(), raw, x[m]);
                    if (!HALF && ZERO) {
                        const u32x4 one = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
                        for (int p = 0; p < PARTS; ++p) ones[m] = mma(T(), x[m][p], one, ones[m]);
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const u32x4 c = codes(T(), w[t][j], hz[t]);
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int p = 0; p < PARTS; ++p) sum[t][m] = mma(T(), x[m][p], c, sum[t][m]);
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float s16 = HALF ? s[t] : 16.f * s[t], sz = s[t] * (8.f - z[t]);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        acc[t][m][q] = fmaf(s16, sum[t][m][q], acc[t][m][q]);
                        if (!HALF && ZERO) acc[t][m][q] = fmaf(sz, ones[m][q], acc[t][m][q]);
                    }
            }
        }
    };

#pragma unroll
    for (int i = 0; i < R - 1; ++i) bring(i);
    for (int i = 0; i < turns; ++i) {
        // run i has landed (loads land in order: all but those of the runs behind it), here and after the barrier for all,
        // and everyone is done with run i - 1, whose place run i + R - 1 takes
        const int behind = min(R - 2, whole - 1 - i);
        if (R > 3 && behind >= 2)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(G::LOADS * 2) : "memory");
        else if (R > 2 && behind >= 1)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(G::LOADS) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        if (NW > 1) asm volatile("s_barrier" ::: "memory");
        bring(i + R - 1);
        if (i < count) consume(i);
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

template <typename T, int NT, int XROWS, int FL, bool S16, bool ZERO, int KW, int NW, int R>
static hipError_t launch(const qcnn_matvec_w4_t &a, hipStream_t s)
{
    typedef W4<T, NT, XROWS, FL, S16, ZERO, KW, NW, R> G;
    const unsigned nblocks = (unsigned)((a.n + 16 * NT * NW - 1) / (16 * NT * NW));
    const unsigned long long blocks = (unsigned long long)nblocks * ((a.rows + XROWS - 1) / XROWS);
    if (blocks * (64 * G::WAVES) > 0xffffffffull) return hipErrorInvalidConfiguration;
    const auto fn = k_w4<T, NT, XROWS, FL, S16, ZERO, KW, NW, R>;
    if (G::LDS > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void *)fn, hipFuncAttributeMaxDynamicSharedMemorySize, G::LDS);
        if (e != hipSuccess) return e;
    }
    fn<<<(unsigned)blocks, 64 * G::WAVES, G::LDS, s>>>(a, nblocks);
    return hipGetLastError();
}

template <typename T, int NT, int XROWS, int FL, int KW, int NW, int R>
static hipError_t run(const qcnn_matvec_w4_t &a, hipStream_t s)
{
    if (a.scale_type != QCNN_F32)
        return a.zero ? launch<T, NT, XROWS, FL, true, true, KW, NW, R>(a, s) : launch<T, NT, XROWS, FL, true, false, KW, NW, R>(a, s);
    return a.zero ? launch<T, NT, XROWS, FL, false, true, KW, NW, R>(a, s) : launch<T, NT, XROWS, FL, false, false, KW, NW, R>(a, s);
}

template <typename T, int FL>
static hipError_t pick_rows(const qcnn_matvec_w4_t &a, hipStream_t s)
{
    constexpr bool F = sizeof(T) == 4;
    if (a.rows > 16) return run<T, 1, F ? 32 : 64, FL, 2, 4, 3>(a, s);
    if (a.rows > 4) return run<T, 1, 16, FL, 2, 4, F ? 3 : 4>(a, s);
    return run<T, 1, 4, FL, 8, 1, FL == 1 ? 3 : 4>(a, s);
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
