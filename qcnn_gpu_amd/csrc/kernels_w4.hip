// Products with 4-bit weights and group scales (qcnn_op_matvec_w4):
//   y[m][j] = sum_g s[g][j] sum_{k in g} (q[j][k] - z[g][j]) x[m][k] + b[j]
//
// Reading the weights is the cost, n * k / 2 bytes; everything else has to keep out of their way.  The codes become
// exact small integers in the type of the matrix instruction (half or bfloat16), 16 x 16 x 32 tiles multiply them with up
// to 16 rows of x at a time, and the group's scale is applied to the float32 sums of the group, one multiplication for
// 32 to 128 weights.  One row of x costs as much as sixteen.
//
// A workgroup owns 16 NT outputs; its waves split k into runs of whole 128s and their sums meet in LDS at the end.  For
// 128 k a lane loads 16 bytes of each of its weight rows: lane l, row l & 15, k from (l >> 4) * 32 on.  Instruction j of
// four wants k = 32 j + (l >> 4) * 8 there, so that its 32 k lie in one group: a 4 x 4 transposition of dwords among the
// lanes l, l + 16, l + 32, l + 48, four swaps of rows of lanes.
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

constexpr int W4_WAVES = 8;

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

// What one wave holds of 128 k: the codes of NT x 16 weight rows, x of MT x 16 rows, the scales (as they stand in memory)
// and zero points of the groups, one for FL instructions.
template <typename T, int NT, int MT, int FL>
struct Stage {
    u32x4 w[NT], x[MT][4][XForm<T>::RAW];
    unsigned s[NT][4 / FL];
    unsigned z[NT][4 / FL];
};

template <typename T, int NT, int MT, int FL, int DEPTH>
__global__ __launch_bounds__(64 * W4_WAVES) void k_w4(const qcnn_matvec_w4_t a, unsigned nblocks)
{
    constexpr int PARTS = XForm<T>::PARTS, RAW = XForm<T>::RAW, VE = sizeof(T) == 4 ? 4 : 8;
    constexpr bool HALF = __is_same(T, f16_t);
    __shared__ float part[W4_WAVES][NT * 256];
    __shared__ __align__(16) uint8_t tail_w[16 * 64];
    __shared__ __align__(16) T tail_x[16 * 128];
    typedef Stage<T, NT, MT, FL> S;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c16 = lane & 15, g = lane >> 4;
    const int n0 = (int)(blockIdx.x % nblocks) * 16 * NT, m0 = (int)(blockIdx.x / nblocks) * 16 * MT;
    const int rows = min(16 * MT, a.rows - m0), row_bytes = (a.k + 1) >> 1;
    // runs of 256 k (a cache line of a weight row), as equal as they can be
    const int units = (a.k + 255) >> 8, blocks = (a.k + 127) >> 7;
    const int kb0 = min(blocks, 2 * (int)((long long)units * wave / W4_WAVES)), kb1 = min(blocks, 2 * (int)((long long)units * (wave + 1) / W4_WAVES));

    const uint8_t *wrow[NT];
    int col[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        col[t] = min(n0 + t * 16 + c16, a.n - 1);
        wrow[t] = (const uint8_t *)a.w + (size_t)col[t] * a.ldw;
    }
    const T *xrow[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) xrow[m] = (const T *)a.x + (size_t)(m0 + min(m * 16 + c16, rows - 1)) * a.ldx;
    const unsigned per = (unsigned)a.group >> 5;

    const auto load_scales = [&](S &st, int kb) {
#pragma unroll
        for (int f = 0; f < 4 / FL; ++f) {
            const int k32 = min(kb * 4 + f * FL, (a.k - 1) >> 5);  // (behind the last group: x is zero there)
            const size_t at = (size_t)((unsigned)k32 / per) * a.n;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                st.s[t][f] = a.scale_type == QCNN_F32 ? ((const unsigned *)a.scale)[at + col[t]] : ((const uint16_t *)a.scale)[at + col[t]];
                st.z[t][f] = a.zero ? ((const uint8_t *)a.zero)[at + col[t]] : 8;
            }
        }
    };
    const auto load = [&](S &st, int kb) {
#pragma unroll
        for (int t = 0; t < NT; ++t) st.w[t] = *(const u32x4_any *)(wrow[t] + (size_t)kb * 64 + g * 16);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int r = 0; r < RAW; ++r) {
                    // of sixteen rows only those that there are ask for x; the others' sums are not stored
                    if (MT > 1 || c16 < rows) st.x[m][j][r] = *(const u32x4_any *)(xrow[m] + kb * 128 + j * 32 + g * 8 + r * 4);
                }
        load_scales(st, kb);
    };
    // The last 128 k where the rows end inside them: x and the codes come through LDS, zeros behind the end of x
    const auto load_tail = [&](S &st, int kb) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            for (int i = g; i < 64; i += 4) tail_w[c16 * 64 + i] = kb * 64 + i < row_bytes ? wrow[t][(size_t)kb * 64 + i] : 0;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            st.w[t] = *(const u32x4 *)(tail_w + c16 * 64 + g * 16);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            T zero;
            from_f32(0.f, zero);
            for (int i = g; i < 128; i += 4) tail_x[c16 * 128 + i] = kb * 128 + i < a.k ? xrow[m][kb * 128 + i] : zero;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int r = 0; r < RAW; ++r) st.x[m][j][r] = *(const u32x4 *)(tail_x + c16 * 128 + j * 32 + g * 8 + r * 4);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        load_scales(st, kb);
    };

    f32x4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[t][m] = f32x4{0, 0, 0, 0};

    const auto compute = [&](const S &st) {
        u32x4 w[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) w[t] = transpose4(st.w[t]);
        f32x4 sum[NT][MT], ones[MT];
#pragma unroll
        for (int f = 0; f < 4 / FL; ++f) {
            if (f) __builtin_amdgcn_sched_barrier(0);  // one group's registers at a time
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                ones[m] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < NT; ++t) sum[t][m] = f32x4{0, 0, 0, 0};
            }
            HalfZero hz[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) hz[t] = half_zero((float)st.z[t][f]);
#pragma unroll
            for (int j = f * FL; j < (f + 1) * FL; ++j) {
                u32x4 x[MT][PARTS];
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    x_operand(T(), st.x[m][j], x[m]);
                    if (!HALF && a.zero) {
                        const u32x4 one = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
                        for (int p = 0; p < PARTS; ++p) ones[m] = mma(T(), x[m][p], one, ones[m]);
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const u32x4 c = codes(T(), w[t][j], hz[t]);
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
#pragma unroll
                        for (int p = 0; p < PARTS; ++p) sum[t][m] = mma(T(), x[m][p], c, sum[t][m]);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const unsigned u = st.s[t][f];
                float s = __uint_as_float(a.scale_type == QCNN_BF16 ? u << 16 : u);
                if (a.scale_type == QCNN_F16) s = (float)__builtin_bit_cast(f16_t, (uint16_t)u);
                const float s16 = HALF ? s : 16.f * s, sz = s * (8.f - (float)st.z[t][f]);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        acc[t][m][i] = fmaf(s16, sum[t][m][i], acc[t][m][i]);
                        if (!HALF && a.zero) acc[t][m][i] = fmaf(sz, ones[m][i], acc[t][m][i]);
                    }
            }
        }
    };

    const bool cut = a.k % 128 != 0 && kb1 == blocks && kb0 < kb1;  // this wave has the end of the rows
    const int whole = kb1 - (cut ? 1 : 0);
    S st[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
        if (MT == 1) {  // lanes without a row keep zeros
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int r = 0; r < RAW; ++r) st[d].x[0][j][r] = u32x4{0, 0, 0, 0};
        }
        if (kb0 + d < whole) load(st[d], kb0 + d);
    }
    for (int kb = kb0; kb < whole; kb += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (kb + d >= whole) break;
            compute(st[d]);
            if (kb + d + DEPTH < whole) load(st[d], kb + d + DEPTH);
        }
    }
    if (cut) {
        load_tail(st[0], whole);
        compute(st[0]);
    }

    // the waves' sums, 16 rows at a time; the lane has rows 4 g .. 4 g + 3 of output c16 of each tile
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        if (m * 16 >= rows) break;
        if (m) __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[wave][(4 * g + i) * (16 * NT) + t * 16 + c16] = acc[t][m][i];
        __syncthreads();
        for (int o = threadIdx.x; o < NT * 256; o += 64 * W4_WAVES) {
            const int row = m * 16 + o / (16 * NT), j = n0 + o % (16 * NT);
            if (row >= rows || j >= a.n) continue;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < W4_WAVES; ++w) v += part[w][o];
            if (a.bias) v += ((const float *)a.bias)[j];
            store_typed(a.y, (size_t)(m0 + row) * a.ldy + j, a.out_type, v);
        }
    }
}

template <typename T, int NT, int MT, int FL, int DEPTH>
static hipError_t run(const qcnn_matvec_w4_t &a, hipStream_t s)
{
    const unsigned nblocks = (unsigned)((a.n + 16 * NT - 1) / (16 * NT));
    const unsigned long long blocks = (unsigned long long)nblocks * ((a.rows + 16 * MT - 1) / (16 * MT));
    if (blocks * (64 * W4_WAVES) > 0xffffffffull) return hipErrorInvalidConfiguration;
    k_w4<T, NT, MT, FL, DEPTH><<<(unsigned)blocks, 64 * W4_WAVES, 0, s>>>(a, nblocks);
    return hipGetLastError();
}

template <typename T, int FL>
static hipError_t pick_rows(const qcnn_matvec_w4_t &a, hipStream_t s)
{
    if (a.rows > 32) return run<T, 2, 4, FL, 1>(a, s);
    if (a.rows > 16) return run<T, 4, 2, FL, 1>(a, s);
    if (a.rows > 4 && a.n > 4096) return run<T, 4, 1, FL, 2>(a, s);
    return run<T, 1, 1, FL, 3>(a, s);
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
