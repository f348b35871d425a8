// 4-bit microscaled factor tables: quantisation, reading back, and the score product.
//
// A row is cut into blocks of 32 elements (the last one padded by zeros).  A block is held as one
// power of two, 2^e with e = floor(log2 max|x|) - 2 in a byte (e + 127), and 32 four-bit codes: a
// sign and one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 (two bits of exponent, one of mantissa), the nearest
// to |x| / 2^e, ties to the even code, anything above 6 as 6.  17 bytes for 32 elements.  A block
// that holds an infinity or a NaN is held as scale byte 255 and reads back as NaN throughout.
#include "alsmi_common.h"
#include "elem.h"

#include <algorithm>
#include <type_traits>

namespace alsmi {

constexpr int MX4_BLOCK = 32;
constexpr int64_t MX4_MAX_WIDTH = 1 << 20;

// 2^(byte - 127) as a float; 255 gives an infinity, which the conversion instructions below take
// as "not a number" for every code of the block.
__device__ __forceinline__ float scale_value(unsigned byte) {
    return __builtin_bit_cast(float, byte ? byte << 23 : 0x00400000u);
}

// ---- quantisation ------------------------------------------------------------------------------
// Scale byte of a block from the bit pattern of its largest |x| (which orders like an unsigned
// integer and puts NaN above infinity above every number).
__device__ __forceinline__ unsigned scale_byte(unsigned max_bits) {
    const unsigned e = max_bits >> 23;  // floor(log2) + 127 (0: below 2^-126)
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
__device__ __forceinline__ unsigned scale_byte(unsigned long long max_bits) {
    const int e = (int)(max_bits >> 52);  // floor(log2) + 1023
    if (e == 2047) return 255u;
    const int b = e - 1023 - 2 + 127;
    return (unsigned)(b < 0 ? 0 : (b > 254 ? 254 : b));
}
__device__ __forceinline__ unsigned abs_bits(float x) {
    return __builtin_bit_cast(unsigned, x) & 0x7fffffffu;
}
__device__ __forceinline__ unsigned long long abs_bits(double x) {
    return __builtin_bit_cast(unsigned long long, x) & 0x7fffffffffffffffull;
}

// The value of another lane of the group that a block shares, as a vector instruction: steps 1 and 2
// exchange within four lanes, then all four agree and step 4 takes the other four's.
template <int STEP>
__device__ __forceinline__ unsigned group_lane(unsigned x) {
    constexpr int CTRL = STEP == 1 ? 0xb1 : STEP == 2 ? 0x4e : 0x141;  // (lane ^ 1, lane ^ 2, mirror of 8)
    return (unsigned)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xf, 0xf, true);
}
template <int STEP>
__device__ __forceinline__ unsigned long long group_lane(unsigned long long x) {
    return ((unsigned long long)group_lane<STEP>((unsigned)(x >> 32)) << 32) |
           group_lane<STEP>((unsigned)x);
}

// E (4 or 8) elements to as many codes, element 0 in the lowest four bits.
template <int E>
__device__ __forceinline__ unsigned to_codes(const float (&x)[E], unsigned byte) {
    const float s = scale_value(byte);
    unsigned c = 0;  // (x / s rounded to nearest even and saturated by the instruction)
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], s, 1);
    if constexpr (E == 8) {
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], s, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], s, 3);
    }
    return byte == 255u ? 0u : c;
}
// fp64 elements are compared with the midpoints in fp64: a first rounding to fp32 could carry a
// value onto a midpoint.
template <int E>
__device__ __forceinline__ unsigned to_codes(const double (&x)[E], unsigned byte) {
    if (byte == 255u) return 0u;
    unsigned c = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const double v = ldexp(fabs(x[i]), 127 - (int)byte);
        unsigned m = (v > 0.25) + (v >= 0.75) + (v > 1.25) + (v >= 1.75) + (v > 2.5) + (v >= 3.5) +
                     (v > 5.0);
        m |= (unsigned)(__builtin_bit_cast(unsigned long long, x[i]) >> 63) << 3;
        c |= m << (4 * i);
    }
    return c;
}

// Elements of T per lane: 16 bytes a load, so that a wave's loads are contiguous.
template <typename T>
constexpr int mx4_lane() {
    return sizeof(T) == 2 ? 8 : 4;
}
// How a workgroup covers rows: `upr` lanes' worth (units) a row, TURNS * 256 units per workgroup, as whole
// rows (`rpb` of them) or as part blockIdx.y of one row.  A launch covers at most MX4_GROUPS workgroups
// of rows (its x extent has to stay below 2^32 threads); the host takes longer tables batch by batch.
constexpr int MX4_TURNS = 4;
constexpr int64_t MX4_GROUPS = (int64_t)1 << 22;
struct RowGrid {
    unsigned upr, rpb, inverse;  // inverse: 2^32 / upr rounded up
    int64_t most;                // rows of a launch
    dim3 grid(int64_t n_rows) const {
        return dim3((unsigned)((n_rows + rpb - 1) / rpb), (upr + 256 * MX4_TURNS - 1) / (256 * MX4_TURNS));
    }
};
static RowGrid row_grid(int nb, int per_lane) {
    RowGrid r;
    constexpr unsigned UNITS = 256 * MX4_TURNS;
    r.upr = (unsigned)nb * (MX4_BLOCK / per_lane);
    r.rpb = r.upr < UNITS ? UNITS / r.upr : 1;
    r.inverse = (unsigned)((((uint64_t)1 << 32) + r.upr - 1) / r.upr);
    r.most = MX4_GROUPS * r.rpb;
    return r;
}
// Row and unit of a thread in a turn; false where there is none.  (x < 1024: the product is exact.)
__device__ __forceinline__ bool row_unit(const unsigned upr, const unsigned rpb, const unsigned inverse,
                                         int turn, int64_t n_rows, int64_t &row, unsigned &sub) {
    const unsigned x = turn * 256 + threadIdx.x;
    const unsigned rl = rpb > 1 ? __umulhi(x, inverse) : 0u;
    sub = x - rl * upr + blockIdx.y * (256 * MX4_TURNS);
    row = (int64_t)blockIdx.x * rpb + rl;
    return rl < rpb && row < n_rows && sub < upr;
}

// Tables larger than the last-level cache go past it: written through it, the lines of one call
// are still being written back during the next (1 M x 128 fp32: reading back 90 us either way, but
// quantising after it 139 us, 101 past the cache).  Smaller ones are left in it for their reader.
constexpr int64_t MX4_STREAM_BYTES = (int64_t)256 << 20;

// A lane takes 16 bytes of elements, 4 or 8 neighbouring lanes a block.  Bound by HBM (1 M x 128 fp32:
// 94 us, 6.2 TB/s).
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(int64_t n_rows, int width,
                                                           const T *__restrict__ x, int64_t ldx,
                                                           uint8_t *__restrict__ codes,
                                                           uint8_t *__restrict__ scales, unsigned upr,
                                                           unsigned rpb, unsigned inverse) {
    typedef typename Elem<T>::wide W;
    constexpr int E = mx4_lane<T>(), LANES = MX4_BLOCK / E;
    typedef typename std::conditional<E == 8, unsigned, unsigned short>::type code_t;
    W v[MX4_TURNS][E];
    int64_t row[MX4_TURNS];
    unsigned sub[MX4_TURNS];
    bool in[MX4_TURNS];
#pragma unroll
    for (int t = 0; t < MX4_TURNS; ++t) {
        in[t] = row_unit(upr, rpb, inverse, t, n_rows, row[t], sub[t]);
        load_n<T, E, STREAM>(v[t], x + (in[t] ? row[t] * ldx + (int64_t)sub[t] * E : 0),
                     in[t] ? width - (int)sub[t] * E : 0);
    }
#pragma unroll
    for (int t = 0; t < MX4_TURNS; ++t) {
        auto m = abs_bits(v[t][0]);
#pragma unroll
        for (int i = 1; i < E; ++i) {
            const auto b = abs_bits(v[t][i]);
            m = b > m ? b : m;
        }
        auto join = [&](auto b) { m = b > m ? b : m; };
        join(group_lane<1>(m));
        join(group_lane<2>(m));
        if constexpr (LANES == 8) join(group_lane<4>(m));
        const unsigned byte = scale_byte(m);
        const unsigned c = to_codes(v[t], byte);
        if (!in[t]) continue;  // (a block's lanes are all in or all out)
        const int64_t at = row[t] * upr + sub[t];
        reinterpret_cast<code_t *>(codes)[at] = (code_t)c;
        if (sub[t] % LANES == 0) scales[at / LANES] = (uint8_t)byte;
    }
}

// ---- reading back --------------------------------------------------------------------------------
template <int E>
__device__ __forceinline__ void from_codes(unsigned c, unsigned byte, float (&v)[E]) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const float s = scale_value(byte);
    const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0);
    const f2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1];
    if constexpr (E == 8) {
        const f2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2);
        const f2 e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
        v[4] = d[0], v[5] = d[1], v[6] = e[0], v[7] = e[1];
    }
}
// (fp64: 6 x 2^127 is past fp32's range, so the scale is applied in fp64)
template <int E>
__device__ __forceinline__ void from_codes(unsigned c, unsigned byte, double (&v)[E]) {
    float f[E];
    from_codes(c, byte == 255u ? 255u : 127u, f);
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = ldexp((double)f[i], (int)byte - 127);
}

// Row i of the output is row rows[i] of the table (row i where rows is null), NaN where there is
// no such row.  Lanes as in mx4_quantize_kernel (1 M x 128 fp32: 82 us, 7.1 TB/s).
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(int64_t n_sel,
                                                             const int32_t *__restrict__ rows,
                                                             int64_t n_rows, int width,
                                                             const uint8_t *__restrict__ codes,
                                                             const uint8_t *__restrict__ scales,
                                                             T *__restrict__ out, int64_t ldo,
                                                             unsigned upr, unsigned rpb,
                                                             unsigned inverse) {
    typedef typename Elem<T>::wide W;
    constexpr int E = mx4_lane<T>(), LANES = MX4_BLOCK / E;
    typedef typename std::conditional<E == 8, unsigned, unsigned short>::type code_t;
    unsigned c[MX4_TURNS], byte[MX4_TURNS];
#pragma unroll
    for (int t = 0; t < MX4_TURNS; ++t) {
        int64_t i;
        unsigned sub;
        c[t] = 0, byte[t] = 255u;
        if (!row_unit(upr, rpb, inverse, t, n_sel, i, sub)) continue;
        const int64_t row = rows ? (int64_t)rows[i] : i;
        if (row < 0 || row >= n_rows) continue;
        const int64_t at = row * upr + sub;
        c[t] = reinterpret_cast<const code_t *>(codes)[at];
        byte[t] = scales[at / LANES];
    }
#pragma unroll
    for (int t = 0; t < MX4_TURNS; ++t) {
        int64_t i;
        unsigned sub;
        if (!row_unit(upr, rpb, inverse, t, n_sel, i, sub)) continue;
        W v[E];
        from_codes(c[t], byte[t], v);
        store_n<T, E, STREAM>(out + i * ldo + (int64_t)sub * E, v, width - (int)sub * E);
    }
}

// ---- scores: out[i, j] = sum_k a[i, k] table[j, k] -----------------------------------------------
// The table's elements have three significant bits and are exact in bf16 once scaled, so the
// product runs on the bf16 matrix cores with fp32 sums (elements of 2^128 and more, scale bytes 253 and
// 254, become infinities there).  The activations are split into bf16 parts: fp32 = 3 parts of 8
// significant bits each (cut, not rounded), fp16 = 2, bf16 = 1.  Bits below bf16's smallest number,
// 2^-133, are cut off; above it the split and every product are exact, and the result has the
// accuracy of fp32 sums of the fp32 products.  (A
// two-way fp16 split as in the half-sweep would take 2 parts for fp32, but needs the table's
// scales applied after each block of 32 and the largest |a| beforehand.)
// Matrix operands: the items are the rows of the result tile, the activations its columns, so a lane
// ends with four consecutive items of one output row.  The contraction index may be spread over
// lane groups and steps in any way both operands share: lane group g takes NBL * 8 consecutive
// elements, one contiguous load of codes and one scale.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Parts;  // bf16 parts of one activation
template <>
struct Parts<float> {
    static constexpr int N = 3;
};
template <>
struct Parts<_Float16> {
    static constexpr int N = 2;
};
template <>
struct Parts<__bf16> {
    static constexpr int N = 1;
};

// upper halves of two floats' bit patterns, the first in the low half
__device__ __forceinline__ unsigned high_halves(float a, float b) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a),
                                 0x07060302u);
}

template <int N, bool FINITE>
__device__ __forceinline__ void split_parts(const float (&x)[8], bf16x8 (&h)[N]) {
    u32x4 w[N];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float a = x[2 * j], b = x[2 * j + 1];
        if constexpr (!FINITE) {  // a NaN keeps a bit in its upper half
            a = a != a ? __builtin_nanf("") : a;
            b = b != b ? __builtin_nanf("") : b;
        }
#pragma unroll
        for (int p = 0; p < N; ++p) {
            w[p][j] = high_halves(a, b);
            if (p + 1 < N) {
                const float ta = __builtin_bit_cast(float, w[p][j] << 16);
                const float tb = __builtin_bit_cast(float, w[p][j] & 0xffff0000u);
                // (an infinity has no further parts)
                a = FINITE || __builtin_isfinite(a) ? a - ta : 0.0f;
                b = FINITE || __builtin_isfinite(b) ? b - tb : 0.0f;
            }
        }
    }
#pragma unroll
    for (int p = 0; p < N; ++p) h[p] = __builtin_bit_cast(bf16x8, w[p]);
}
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&h)[N]) {
    if constexpr (N == 1) {
        split_parts<1, true>(x, h);  // (bf16 as it is)
    } else {
        // the tests for infinities and NaN are half of the work: one test for all eight
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned b = __builtin_bit_cast(unsigned, x[i]) & 0x7fffffffu;
            top = b > top ? b : top;
        }
        if (__any(top >= 0x7f800000u)) split_parts<N, false>(x, h);
        else split_parts<N, true>(x, h);
    }
}

// eight codes to bf16
__device__ __forceinline__ bf16x8 codes_to_bf16(unsigned c, float s) {
    u32x4 w;
    w[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0));
    w[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1));
    w[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2));
    w[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3));
    return __builtin_bit_cast(bf16x8, w);
}

// NW words of codes; a block behind the row's end is zero
template <int NW>
__device__ __forceinline__ void load_codes(unsigned (&c)[NW], const uint8_t *p) {
    typedef unsigned vec_t __attribute__((ext_vector_type(NW), aligned(4)));
    if constexpr (NW == 1) {
        c[0] = *reinterpret_cast<const unsigned *>(p);
    } else {
        const vec_t v = *reinterpret_cast<const vec_t *>(p);
#pragma unroll
        for (int i = 0; i < NW; ++i) c[i] = v[i];
    }
}

// The activations of a call: their rows may be picked out of a larger table.
struct Rows {
    int64_t n_sel, n_rows, ld;
    const int32_t *ids;  // null: row i is row i
    // row of selected row i, or -1 where there is none
    __device__ __forceinline__ int64_t of(int64_t i) const {
        const int64_t r = ids ? (int64_t)ids[i] : i;
        return r >= 0 && r < n_rows ? r : -1;
    }
};

struct ScoreStore {
    void *out;
    int64_t ld, n_sel, n_items;
};
// Row i of a wave's tile n is item item_of<TO>(n, i) of its 16 NT items, so that a store of 16 bytes per
// lane (group g) leaves the four groups' side by side, 64 bytes of a score row: fp32 tiles as they
// come, 16-bit ones in pairs, where a lane holds eight consecutive items.  (With 4 NT consecutive
// items per lane, every store a quarter or half of each line it touches, 2048 x 16384 x 4096 bf16
// took 94 us instead of 79, 512 x 26744 x 64 fp32 20.7 instead of 18.3.)
template <typename TO>
__device__ __forceinline__ int item_of(int n, int i) {
    return sizeof(TO) == 4 ? 16 * n + i : (n >> 1) * 32 + (i >> 2) * 8 + (n & 1) * 4 + (i & 3);
}
// Group g's part of one output row from the NT tiles' results v[n]; `item` is the wave's first.
template <typename TO, int NT>
__device__ __forceinline__ void put_row(TO *row, int64_t item, int g, int64_t n_items,
                                        const f32x4 (&v)[NT]) {
    static_assert(NT % 2 == 0, "tiles in pairs");
    typedef TO vec_t __attribute__((ext_vector_type(16 / sizeof(TO)), aligned(sizeof(TO))));
    if (!row) return;
    if (item + 16 * NT <= n_items) {
        TO *p = row + item + item_of<TO>(0, 4 * g);
        if constexpr (sizeof(TO) == 4) {
#pragma unroll
            for (int n = 0; n < NT; ++n) *reinterpret_cast<vec_t *>(p + 16 * n) = v[n];
        } else {
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
                vec_t w;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = (TO)v[n][i], w[4 + i] = (TO)v[n + 1][i];
                *reinterpret_cast<vec_t *>(p + 16 * n) = w;
            }
        }
    } else {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t at = item + item_of<TO>(n, 4 * g + i);
                if (at < n_items) row[at] = (TO)v[n][i];
            }
    }
}
template <typename TO>
__device__ __forceinline__ TO *out_row(const ScoreStore &o, int64_t row) {
    return row < o.n_sel ? static_cast<TO *>(o.out) + row * o.ld : nullptr;
}

// Rows of at most eight blocks (rank <= 128: four): UT tiles of 16 activation rows stay in registers,
// split once, and the wave walks `tpw` tiles of 16 items.  Bound by the table's bytes for a few
// rows (1 x 1000000 x 128 bf16: 13.2 us, 5.4 TB/s), by the write of the scores for many (512 x 26744
// x 64 fp32: 18.3 us, 11 without it).
template <typename T, typename TO, int NBL, int UT, int NT>
__global__ __launch_bounds__(256) void mx4_scores_narrow_kernel(Rows rows, const T *__restrict__ a,
                                                                int width,
                                                                const uint8_t *__restrict__ codes,
                                                                const uint8_t *__restrict__ scales,
                                                                int nb, ScoreStore o, int groups,
                                                                int tpw) {
    constexpr int NP = Parts<T>::N;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int g = lane >> 4, q = lane & 15;
    const unsigned chunk = blockIdx.x / (unsigned)groups;
    const int64_t row_base = (int64_t)(blockIdx.x - chunk * groups) * (16 * UT);
    const int64_t n_tiles = (o.n_items + 15) / 16;
    const int64_t t0 = ((int64_t)chunk * 4 + wave) * tpw;
    const int64_t t1 = t0 + tpw < n_tiles ? t0 + tpw : n_tiles;
    constexpr int BL = NBL > 4 ? NBL / 4 : 1;  // blocks of a lane
    const int blk = (g * NBL) >> 2;            // the first of them
    // NT neighbouring tiles per turn: a lane's stores of one output row lie side by side.  The codes
    // of the next turn are on their way during the products of this one.
    unsigned c[NT][NBL];
    unsigned sb[NT][BL];
    auto fetch = [&](int64_t tile) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            int64_t item = 16 * tile + item_of<TO>(n, q);
            item = item < o.n_items ? item : o.n_items - 1;
            const uint8_t *from = codes + item * (16 * (int64_t)nb) + g * NBL * 4;
#pragma unroll
            for (int j = 0; j < NBL; ++j) c[n][j] = 0;
#pragma unroll
            for (int l = 0; l < BL; ++l) {
                sb[n][l] = 127u;
                if (blk + l >= nb) continue;
                constexpr int W = NBL > 4 ? 4 : NBL;
                load_codes<W>(*reinterpret_cast<unsigned(*)[W]>(&c[n][l * 4]), from + 16 * l);
                sb[n][l] = scales[item * nb + blk + l];
            }
        }
    };
    if (t0 < t1) fetch(t0);
    // the four waves split a quarter of the activations each and hand them round through LDS
    __shared__ bf16x8 shared_a[UT * NBL][NP][64];
#pragma unroll
    for (int f = 0; f < UT * NBL; f += 4) {
        const int part = f + wave;
        if (UT * NBL >= 4 || part < UT * NBL) {
            const int t = part / NBL, j = part - t * NBL;
            int64_t i = row_base + 16 * t + q;
            i = i < rows.n_sel ? i : rows.n_sel - 1;  // (rows past the end are not stored)
            const int64_t r = rows.of(i);
            const int k = (g * NBL + j) * 8;
            float x[8];
            load8<T>(x, a + (r < 0 ? 0 : r) * rows.ld + k, width - k);
            if (r < 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = __builtin_nanf("");
            }
            bf16x8 h[NP];
            split8<NP>(x, h);
#pragma unroll
            for (int p = 0; p < NP; ++p) shared_a[part][p][lane] = h[p];
        }
    }
    __syncthreads();
    if (t0 >= t1) return;
    bf16x8 af[UT][NBL][NP];
#pragma unroll
    for (int t = 0; t < UT; ++t)
#pragma unroll
        for (int j = 0; j < NBL; ++j)
#pragma unroll
            for (int p = 0; p < NP; ++p) af[t][j][p] = shared_a[t * NBL + j][p][lane];
    TO *dst[UT];
#pragma unroll
    for (int t = 0; t < UT; ++t) dst[t] = out_row<TO>(o, row_base + 16 * t + q);
    for (int64_t tile = t0; tile < t1; tile += NT) {
        bf16x8 b[NT][NBL];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < NBL; ++j) b[n][j] = codes_to_bf16(c[n][j], scale_value(sb[n][j / 4]));
        if (tile + NT < t1) fetch(tile + NT);
        f32x4 acc[UT][NT];
#pragma unroll
        for (int t = 0; t < UT; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[t][n] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < NBL; ++j)
#pragma unroll
            for (int p = NP - 1; p >= 0; --p)  // small parts first
#pragma unroll
                for (int t = 0; t < UT; ++t)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        acc[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[n][j], af[t][j][p],
                                                                            acc[t][n], 0, 0, 0);
#pragma unroll
        for (int t = 0; t < UT; ++t)
            put_row<TO, NT>(dst[t], 16 * tile, g, o.n_items, acc[t]);
    }
}

// Sums the KW waves' tiles into wave 0's, in wave order; whether this wave holds the result.
template <int MT, int NT, int KW>
__device__ __forceinline__ bool join_waves(f32x4 (&acc)[MT][NT], int wave, int lane) {
    if constexpr (KW > 1) {
        __shared__ f32x4 part[KW - 1][MT * NT][64];
        if (wave > 0) {
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int n = 0; n < NT; ++n) part[wave - 1][t * NT + n][lane] = acc[t][n];
        }
        __syncthreads();
        if (wave > 0) return false;
#pragma unroll
        for (int w = 0; w < KW - 1; ++w)
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[t][n] += part[w][t * NT + n][lane];
    }
    return true;
}

// Rows of any width: a wave forms MT x NT tiles (16 activation rows x 16 items each) in steps of
// four blocks.  KW = 1: the four waves of a workgroup take neighbouring items; KW = 4: they share
// one tile group and take a quarter of the steps each, joined in wave order through LDS, where
// there are too few tiles to fill the chip.  Bound by the loads of each step for a few rows (none is in
// flight across steps; 1 x 1000000 x 512 bf16: 90 us, 3 TB/s of table), by the loads and splits of
// the activations else.
template <typename T, typename TO, int MT, int NT, int KW>
__global__ __launch_bounds__(256) void mx4_scores_wide_kernel(Rows rows, const T *__restrict__ a,
                                                              int width,
                                                              const uint8_t *__restrict__ codes,
                                                              const uint8_t *__restrict__ scales,
                                                              int nb, ScoreStore o, int groups) {
    constexpr int NP = Parts<T>::N;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int g = lane >> 4, q = lane & 15;
    const unsigned chunk = blockIdx.x / (unsigned)groups;
    const int64_t row_base = (int64_t)(blockIdx.x - chunk * groups) * (16 * MT);
    const int64_t item_base = (KW == 1 ? (int64_t)chunk * 4 + wave : (int64_t)chunk) * (16 * NT);
    const int steps = (nb + 3) / 4;
    int s0 = 0, s1 = steps;
    if constexpr (KW > 1) {
        const int per = (steps + KW - 1) / KW;
        s0 = wave * per < steps ? wave * per : steps;
        s1 = s0 + per < steps ? s0 + per : steps;
    }
    const T *ar[MT];
    bool no_row[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        int64_t i = row_base + 16 * t + q;
        i = i < rows.n_sel ? i : rows.n_sel - 1;
        const int64_t r = rows.of(i);
        no_row[t] = r < 0;
        ar[t] = a + (r < 0 ? 0 : r) * rows.ld;
    }
    int64_t it[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int64_t i = item_base + item_of<TO>(n, q);
        it[n] = i < o.n_items ? i : o.n_items - 1;
    }
    f32x4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[t][n] = f32x4{0, 0, 0, 0};
    if (item_base < o.n_items) {
        for (int s = s0; s < s1; ++s) {
            const int blk = 4 * s + g;
            unsigned c[NT][4];
            float sc[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                sc[n] = 1.0f;
#pragma unroll
                for (int j = 0; j < 4; ++j) c[n][j] = 0;
                if (blk < nb) {
                    load_codes<4>(c[n], codes + (it[n] * nb + blk) * 16);
                    sc[n] = scale_value(scales[it[n] * nb + blk]);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = blk * 32 + 8 * j;
                bf16x8 b[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) b[n] = codes_to_bf16(c[n][j], sc[n]);
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    float x[8];
                    load8<T>(x, ar[t] + k, width - k);
                    bf16x8 h[NP];
                    split8<NP>(x, h);
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            acc[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[n], h[p], acc[t][n],
                                                                                0, 0, 0);
                }
            }
        }
    }
    if (!join_waves<MT, NT, KW>(acc, wave, lane)) return;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        if (no_row[t]) {
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[t][n] = f32x4{} + __builtin_nanf("");
        }
        put_row<TO, NT>(out_row<TO>(o, row_base + 16 * t + q), item_base, g, o.n_items, acc[t]);
    }
}

// ---- loads straight into LDS ---------------------------------------------------------------------
// 16 bytes per lane from `bytes` behind `from` + `offset` (both the same for the whole wave) to the
// wave's 1024 bytes at `to`, lane by lane.  Through a buffer descriptor and not by address: while a
// load of the latter kind is in flight the compiler lets every read of LDS wait for all reads before
// it (2048 x 16384 x 4096 79 us instead of 76).
typedef __amdgpu_buffer_rsrc_t buffer_t;
__device__ __forceinline__ buffer_t buffer_of(const void *from) {
    constexpr int DATA_32 = 4 << 15;  // (4 GiB of 32-bit words, no stride)
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(from), 0, -1, DATA_32);
}
__device__ __forceinline__ void load_to_lds(buffer_t from, unsigned offset, unsigned bytes, u32x4 *to) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)to, 16,
                                             (int)bytes, (int)offset, 0, 0);
}

// ---- large products of float activations ---------------------------------------------------------
// A first kernel splits the activations into their bf16 parts, rows picked and padded to whole turns
// (planes[p][row][steps * 64]); a second one forms 128 rows x 64 WN items per workgroup through LDS,
// 2 WN waves of 64 x 64, in steps of 64 elements, two steps a turn.  Parts and codes go from
// memory straight into LDS, into two buffers; the codes become bf16 in registers, once per wave
// and step for all parts of 64 rows.  Each part costs one matrix instruction: fp32 activations run at a
// third of the bf16 rate (2000 x 16000 x 2000: bf16 156 us, 0.82 PFLOP/s, fp16 255, fp32 338, 1.15 counted
// by parts).  Bound by the loads of the parts (without them bf16 116, fp16 185, fp32 of WN = 2 336 instead
// of 447; a third buffer changes nothing).
constexpr int WT_ROWS = 128, WT_ITEMS = 128;
constexpr int64_t MX4_SPLIT_BYTES = (int64_t)256 << 20;  // of parts at a time

template <typename T>
__global__ __launch_bounds__(256) void mx4_split_kernel(Rows rows, const T *__restrict__ a, int width,
                                                        int units, u32x4 *__restrict__ planes) {
    constexpr int NP = Parts<T>::N;
    const int64_t i = blockIdx.x;  // one row per workgroup, eight elements per thread and turn
    const int64_t r = rows.of(i);
    for (int u = threadIdx.x; u < units; u += 256) {
        float x[8];
        load8<T>(x, a + (r < 0 ? 0 : r) * rows.ld + (int64_t)u * 8, width - u * 8);
        if (r < 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __builtin_nanf("");
        }
        bf16x8 h[NP];
        split8<NP>(x, h);
#pragma unroll
        for (int p = 0; p < NP; ++p)
            planes[((int64_t)p * rows.n_sel + i) * units + u] = __builtin_bit_cast(u32x4, h[p]);
    }
}

template <typename TO, int NP, int WN>
__global__ __launch_bounds__(128 * WN, NP > 2 && WN == 2 ? 1 : 2) void mx4_scores_split_kernel(
    const u32x4 *__restrict__ planes, const uint8_t *__restrict__ codes,
    const uint8_t *__restrict__ scales, int nb, ScoreStore o, int row_tiles) {
    constexpr int MT = 4, NT = 4, THREADS = 128 * WN, ITEMS = 64 * WN;
    constexpr int LA = WT_ROWS * 8 / THREADS;  // 16-byte loads per thread, part and step
    static_assert(ITEMS * 2 == THREADS, "one block of codes per thread and step");
    // rows of the parts (eight chunks of eight elements each, permuted as in mx4_scores_tiled_kernel)
    // and of the items (two blocks each); separate arrays: see there
    __shared__ u32x4 sa0[NP * WT_ROWS * 8], sa1[NP * WT_ROWS * 8];
    __shared__ u32x4 sb0[ITEMS * 2], sb1[ITEMS * 2];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, q = lane & 15;
    const unsigned total = gridDim.x, xcd = blockIdx.x & 7u, nth = blockIdx.x >> 3;
    const unsigned per = total >> 3, extra = total & 7u;
    const unsigned tile = xcd * per + (xcd < extra ? xcd : extra) + nth;
    const int64_t row_base = (int64_t)(tile % (unsigned)row_tiles) * WT_ROWS;
    const int64_t item_base = (int64_t)(tile / (unsigned)row_tiles) * ITEMS;
    const int turns = (nb + 3) / 4;
    const int64_t units = (int64_t)turns * 16;  // chunks of a row of the planes
    auto b_row = [&](int i) {
        const int64_t r = item_base + i;
        return r < o.n_items ? r : o.n_items - 1;
    };
    // A thread's slots in a part's rows: row THREADS / 8 i + tid / 8, chunk (tid % 8) ^ (row / 2 % 8), the same
    // for every i; its slot of the items: place tid / 2, block tid % 2.  The item at a place: the 16
    // items that a matrix operand reads at once lie side by side.
    const int chunk = (tid & 7) ^ (tid >> 4 & 7);
    // (in bytes: the parts of a call take less than 4 GiB, a tile's codes 128 MiB at most)
    const buffer_t a_mem = buffer_of(planes), b_mem = buffer_of(codes + item_base * nb * 16);
    unsigned asrc[LA];
#pragma unroll
    for (int i = 0; i < LA; ++i) {
        const int64_t r = row_base + i * (THREADS / 8) + (tid >> 3);
        asrc[i] = (unsigned)((r < o.n_sel ? r : o.n_sel - 1) * units + chunk) * 16u;
    }
    const unsigned plane = (unsigned)(o.n_sel * units) * 16u;
    const int place = tid >> 1;
    const unsigned bsrc =
        (unsigned)(b_row((place & ~63) + item_of<TO>(place >> 4 & 3, place & 15)) - item_base) * (unsigned)nb;
    auto load_step = [&](unsigned step, u32x4 *to_a, u32x4 *to_b) __attribute__((always_inline)) {
        // (one step is loaded past the last turn, and not used)
        const unsigned s = step < 2u * turns ? step : 0u;
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int i = 0; i < LA; ++i)
                load_to_lds(a_mem, p * plane + s * 128u, asrc[i],
                            &to_a[(p * LA + i) * THREADS + wave * 64]);
        // (a block behind the row's end meets zeros of the activations: any codes will do)
        const unsigned k = 2u * s + (tid & 1);
        load_to_lds(b_mem, 0, (bsrc + (k < (unsigned)nb ? k : nb - 1)) * 16u, &to_b[wave * 64]);
    };
    const int wm = wave & 1, wn = wave >> 1;
    const int ar = wm * 64 + q, sa = ar >> 1 & 7;
    const uint8_t *srow[NT];  // the scales of this lane's items
#pragma unroll
    for (int n = 0; n < NT; ++n) srow[n] = scales + b_row(wn * 64 + item_of<TO>(n, q)) * nb;
    unsigned sw[NT];
    auto load_scales = [&](int turn) {  // the turn's four scales; 1 behind the row's end
        typedef unsigned word_t __attribute__((aligned(1)));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (4 * turn + 4 <= nb) {
                sw[n] = *reinterpret_cast<const word_t *>(srow[n] + 4 * turn);
            } else {
                sw[n] = 0x7f7f7f7fu;
                for (int i = 0; 4 * turn + i < nb; ++i)
                    sw[n] = (sw[n] & ~(255u << (8 * i))) | (unsigned)srow[n][4 * turn + i] << (8 * i);
            }
        }
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[t][n] = f32x4{0, 0, 0, 0};
    auto products = [&](int step, const u32x4 *a, const u32x4 *b, const unsigned (&w)[NT])
                        __attribute__((always_inline)) {
        const u32x2 *codes_of = reinterpret_cast<const u32x2 *>(b) + (wn * 64 + q) * 4 + g;
        u32x2 c[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) c[n] = codes_of[n * 16 * 4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            bf16x8 bf[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n)
                bf[n] = codes_to_bf16(c[n][j], scale_value(w[n] >> (16 * step + 8 * (g >> 1)) & 255u));
#pragma unroll
            for (int p = NP - 1; p >= 0; --p)
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const bf16x8 af = __builtin_bit_cast(
                        bf16x8, a[(p * WT_ROWS + ar + 16 * t) * 8 + ((2 * g + j) ^ sa)]);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        acc[t][n] =
                            __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[n], af, acc[t][n], 0, 0, 0);
                }
        }
    };
    load_scales(0);
    load_step(0, sa0, sb0);
    for (int turn = 0; turn < turns; ++turn) {
        unsigned w[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) w[n] = sw[n];
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's part of the step is in LDS
        __syncthreads();                     // everyone's is, and the other buffer is free
        load_step(2 * turn + 1, sa1, sb1);
        if (turn + 1 < turns) load_scales(turn + 1);
        __builtin_amdgcn_sched_barrier(0);
        products(0, sa0, sb0, w);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0x0f70);
        __syncthreads();
        load_step(2 * turn + 2, sa0, sb0);
        __builtin_amdgcn_sched_barrier(0);
        products(1, sa1, sb1, w);
        __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);  // (the step loaded for nothing)
#pragma unroll
    for (int t = 0; t < MT; ++t)
        put_row<TO, NT>(out_row<TO>(o, row_base + ar + 16 * t), item_base + wn * 64, g, o.n_items,
                        acc[t]);
}

// Both sides in 4 bits: v_mfma_scale_f32_16x16x128_f8f6f4 takes 32 codes per lane (one block) and
// its scale byte, four blocks per instruction.
__device__ __forceinline__ i32x8 as_operand(u32x4 w) {
    return i32x8{(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
}
// Block `blk` of a row, or zeros with scale 1 behind the row's end.
__device__ __forceinline__ void load_block(const uint8_t *__restrict__ c, const uint8_t *__restrict__ s,
                                           int64_t row, int blk, int nb, u32x4 &w, int &e) {
    typedef unsigned vec_t __attribute__((ext_vector_type(4), aligned(4)));
    w = u32x4{0, 0, 0, 0};
    e = 127;
    if (blk < nb) {
        w = *reinterpret_cast<const vec_t *>(c + (row * nb + blk) * 16);
        e = s[row * nb + blk];
    }
}

// Rows of at most 4 NS blocks: the activations stay in registers and the wave walks the items, as in
// mx4_scores_narrow_kernel (1 x 1000000 x 200: 20 us, 6.0 TB/s; 2000 x 26744 x 200 fp32 48).
template <typename TO, int NS, int UT, int NT>
__global__ __launch_bounds__(256) void mx4_scores_both_narrow_kernel(
    Rows rows, const uint8_t *__restrict__ acodes, const uint8_t *__restrict__ ascales,
    const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, int nb, ScoreStore o,
    int groups, int tpw) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int g = lane >> 4, q = lane & 15;
    const unsigned chunk = blockIdx.x / (unsigned)groups;
    const int64_t row_base = (int64_t)(blockIdx.x - chunk * groups) * (16 * UT);
    const int64_t n_tiles = (o.n_items + 15) / 16;
    const int64_t t0 = ((int64_t)chunk * 4 + wave) * tpw;
    const int64_t t1 = t0 + tpw < n_tiles ? t0 + tpw : n_tiles;
    if (t0 >= t1) return;
    u32x4 c[NT][NS];
    int e[NT][NS];
    auto fetch = [&](int64_t tile) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            int64_t item = 16 * tile + item_of<TO>(n, q);
            item = item < o.n_items ? item : o.n_items - 1;
#pragma unroll
            for (int s = 0; s < NS; ++s)
                load_block(codes, scales, item, 4 * s + g, nb, c[n][s], e[n][s]);
        }
    };
    fetch(t0);
    u32x4 aw[UT][NS];
    int ae[UT][NS];
    TO *dst[UT];
#pragma unroll
    for (int t = 0; t < UT; ++t) {
        const int64_t i = row_base + 16 * t + q;
        const int64_t r = rows.of(i < rows.n_sel ? i : rows.n_sel - 1);
        dst[t] = out_row<TO>(o, i);
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            load_block(acodes, ascales, r < 0 ? 0 : r, 4 * s + g, nb, aw[t][s], ae[t][s]);
            if (r < 0) ae[t][s] = 255;  // no such row: NaN
        }
    }
    for (int64_t tile = t0; tile < t1; tile += NT) {
        f32x4 acc[UT][NT];
#pragma unroll
        for (int t = 0; t < UT; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[t][n] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int t = 0; t < UT; ++t)
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    acc[t][n] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        as_operand(c[n][s]), as_operand(aw[t][s]), acc[t][n], 4, 4, 0, e[n][s], 0,
                        ae[t][s]);
        if (tile + NT < t1) fetch(tile + NT);
#pragma unroll
        for (int t = 0; t < UT; ++t)
            put_row<TO, NT>(dst[t], 16 * tile, g, o.n_items, acc[t]);
    }
}

// Any width, straight from memory: the form for a few rows and for products too small to tile.  KW as
// in mx4_scores_wide_kernel (1 x 1000000 x 512: 48 us, 5.7 TB/s).
template <typename TO, int MT, int NT, int KW>
__global__ __launch_bounds__(256) void mx4_scores_both_kernel(Rows rows,
                                                              const uint8_t *__restrict__ acodes,
                                                              const uint8_t *__restrict__ ascales,
                                                              const uint8_t *__restrict__ codes,
                                                              const uint8_t *__restrict__ scales,
                                                              int nb, ScoreStore o, int groups) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int g = lane >> 4, q = lane & 15;
    const unsigned chunk = blockIdx.x / (unsigned)groups;
    const int64_t row_base = (int64_t)(blockIdx.x - chunk * groups) * (16 * MT);
    const int64_t item_base = (KW == 1 ? (int64_t)chunk * 4 + wave : (int64_t)chunk) * (16 * NT);
    if (item_base >= o.n_items) return;  // (with KW > 1 no workgroup has only some such waves)
    int64_t ai[MT], it[NT];
    bool no_row[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        int64_t i = row_base + 16 * t + q;
        i = i < rows.n_sel ? i : rows.n_sel - 1;
        const int64_t r = rows.of(i);
        no_row[t] = r < 0;
        ai[t] = r < 0 ? 0 : r;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int64_t i = item_base + item_of<TO>(n, q);
        it[n] = i < o.n_items ? i : o.n_items - 1;
    }
    f32x4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[t][n] = f32x4{0, 0, 0, 0};
    const int steps = (nb + 3) / 4, per = (steps + KW - 1) / KW;
    const int s0 = KW == 1 ? 0 : wave * per, s1 = s0 + per < steps ? s0 + per : steps;
    for (int s = s0; s < s1; ++s) {
        const int blk = 4 * s + g;
        u32x4 af[MT], bf[NT];
        int as[MT], bs[NT];
#pragma unroll
        for (int t = 0; t < MT; ++t) load_block(acodes, ascales, ai[t], blk, nb, af[t], as[t]);
#pragma unroll
        for (int n = 0; n < NT; ++n) load_block(codes, scales, it[n], blk, nb, bf[n], bs[n]);
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n)
                acc[t][n] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                    as_operand(bf[n]), as_operand(af[t]), acc[t][n], 4, 4, 0, bs[n], 0, as[t]);
    }
    if (!join_waves<MT, NT, KW>(acc, wave, lane)) return;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        if (no_row[t]) {
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[t][n] = f32x4{} + __builtin_nanf("");
        }
        put_row<TO, NT>(out_row<TO>(o, row_base + 16 * t + q), item_base, g, o.n_items, acc[t]);
    }
}

// The same for large products, tiled through LDS: a workgroup of WM x WN waves forms BM rows x BN
// items in steps of eight blocks (128 bytes a row), two steps a turn, each wave MT x NT tiles of
// 16 x 16.
//  - Codes go from memory straight into LDS (16 bytes per lane), into two buffers: the next step's are on
//    their way during this step's products.  The chunks of a row lie permuted, so the 16 rows
//    that a matrix operand reads at once spread over all banks.
//  - Lane group g takes blocks 2g and 2g + 1 of a step (the contraction index may be dealt out in
//    any way both sides share): one word brings their scales for both steps of the turn, and the
//    instruction picks the byte.  Scales go through registers, 16 of a row at a time, one turn ahead.
//  - A turn has no branch in it: otherwise the compiler moves products behind the next barrier and
//    keeps all their operands.  The blocks of a row behind the last whole turn are read from memory.
//  - An operand is needed every MT products; the reads are spread between them by hand.
// Workgroups are dealt to the eight XCDs in contiguous ranges, so that neighbours in a cache
// share their operands.  2048 x 16384 x 4096 -> bf16 74 us, 3.7 PFLOP/s; the matrix instructions alone
// 54 us, the reads of LDS and the loads into it some 10 more, the stores the rest.
template <typename TO, int WM, int WN, int MT, int NT>
__global__ __launch_bounds__(64 * WM * WN, 2) void mx4_scores_tiled_kernel(
    Rows rows, const uint8_t *__restrict__ acodes, const uint8_t *__restrict__ ascales,
    const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, int nb, ScoreStore o,
    int row_tiles) {
    constexpr int THREADS = 64 * WM * WN;
    constexpr int BM = WM * MT * 16, BN = WN * NT * 16;
    static_assert(BM + BN == THREADS, "one row of scales per thread");
    constexpr int LA = BM * 8 / THREADS, LB = BN * 8 / THREADS;  // 16-byte loads per thread and step
    // rows of the activations, then of the items; two arrays and not one of two halves: only for
    // different arrays does the compiler see that a read of one need not wait for the loads into
    // the other
    __shared__ u32x4 sc0[(BM + BN) * 8], sc1[(BM + BN) * 8];
    __shared__ u32x4 ss[2][BM + BN];  // word g of a row: the scales for lane group g in a turn
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // (in a scalar register)
    const int g = lane >> 4, q = lane & 15;
    // contiguous ranges of tiles per XCD (workgroups are dealt out to them in turn)
    const unsigned total = gridDim.x, xcd = blockIdx.x & 7u, nth = blockIdx.x >> 3;
    const unsigned per = total >> 3, extra = total & 7u;
    const unsigned tile = xcd * per + (xcd < extra ? xcd : extra) + nth;
    const int64_t row_base = (int64_t)(tile % (unsigned)row_tiles) * BM;
    const int64_t item_base = (int64_t)(tile / (unsigned)row_tiles) * BN;
    auto a_row = [&](int i) {  // table row of the tile's row i (some row where there is none)
        int64_t r = row_base + i;
        r = rows.of(r < rows.n_sel ? r : rows.n_sel - 1);
        return r < 0 ? 0 : r;
    };
    auto b_row = [&](int i) {
        const int64_t r = item_base + i;
        return r < o.n_items ? r : o.n_items - 1;
    };
    // slot s of a buffer: row s / 8, chunk (s % 8) ^ swizzle of the row; a thread's slots are THREADS
    // apart, THREADS / 8 rows, which leaves the swizzles as they are
    auto a_swz = [](unsigned row) { return row >> 1 & 7u; };
    auto b_swz = [](unsigned row) {  // (rows as item_of deals them to 16 lanes)
        return sizeof(TO) == 4 ? row >> 1 & 7u : (row >> 1 & 1u) | (row >> 3 & 3u) << 1;
    };
    static_assert(THREADS / 8 % 32 == 0, "rows between a thread's slots");
    const unsigned ca = (tid & 7) ^ a_swz(tid >> 3), cb = (tid & 7) ^ b_swz(tid >> 3);
    // bytes of the thread's chunk of a step from the tile's first row on (from the table's where rows are
    // picked: the host makes sure that 32 bits do)
    const int64_t a_first = rows.ids ? 0 : row_base;
    const buffer_t a_mem = buffer_of(acodes + a_first * nb * 16),
                   b_mem = buffer_of(codes + item_base * nb * 16);
    unsigned src[LA + LB];
#pragma unroll
    for (int i = 0; i < LA + LB; ++i) {
        const int row = (i < LA ? i : i - LA) * (THREADS / 8) + (tid >> 3);
        src[i] = i < LA ? ((unsigned)(a_row(row) - a_first) * (unsigned)nb + ca) * 16u
                        : ((unsigned)(b_row(row) - item_base) * (unsigned)nb + cb) * 16u;
    }
    const int turns = nb / 16;
    auto load_step = [&](unsigned step, u32x4 *to) __attribute__((always_inline)) {
        // (one step is loaded past the last turn, and not used)
        const unsigned s = step < 2u * turns ? step : 0u;
#pragma unroll
        for (int i = 0; i < LA + LB; ++i)
            load_to_lds(i < LA ? a_mem : b_mem, s * 128u, src[i], &to[i * THREADS + wave * 64]);
    };
    const uint8_t *scale_row = tid < BM ? ascales + a_row(tid) * nb : scales + b_row(tid - BM) * nb;
    typedef unsigned unaligned_t __attribute__((ext_vector_type(4), aligned(1)));
    f32x4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[t][n] = f32x4{0, 0, 0, 0};
    const int wm = wave % WM, wn = wave / WM;
    // rows in the buffers
    const int ar = wm * MT * 16 + q;
    const int br = wn * NT * 16 + item_of<TO>(0, q);
    const int sa = a_swz(ar), sb = b_swz(br);  // (the same for all of the wave's tiles)
    // the products of one step; SECOND: of the second step of a turn
    auto products = [&](auto second, const u32x4 *buf, const int (&as)[MT], const int (&bs)[NT])
                        __attribute__((always_inline)) {
        constexpr int S = 2 * decltype(second)::value;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            i32x8 af[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t)
                af[t] = as_operand(buf[(ar + 16 * t) * 8 + ((2 * g + h) ^ sa)]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const i32x8 bf = as_operand(buf[(BM + br + item_of<TO>(n, 0)) * 8 + ((2 * g + h) ^ sb)]);
#pragma unroll
                for (int t = 0; t < MT; ++t)
                    acc[t][n] = h == 0 ? __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                                             bf, af[t], acc[t][n], 4, 4, S, bs[n], S, as[t])
                                       : __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                                             bf, af[t], acc[t][n], 4, 4, S + 1, bs[n], S + 1, as[t]);
            }
        }
    };
    // order of the above: first the reads of the scales, the first half's activations and two
    // items' codes; then one read of the item operand two turns ahead before every MT products, the
    // second half's activations in the last two turns of the first
    auto spread = [&](auto extra) __attribute__((always_inline)) {
        constexpr int DS_READ = 0x100, MFMA = 0x8;
        __builtin_amdgcn_sched_group_barrier(DS_READ, decltype(extra)::value + MT + 2, 0);
#pragma unroll
        for (int n = 0; n < 2 * NT; ++n) {
            __builtin_amdgcn_sched_group_barrier(MFMA, MT, 0);
            if (n == NT - 2 || n == NT - 1) __builtin_amdgcn_sched_group_barrier(DS_READ, MT / 2 + 1, 0);
            else if (n < 2 * NT - 2) __builtin_amdgcn_sched_group_barrier(DS_READ, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    if (turns > 0) {
        u32x4 sr = *reinterpret_cast<const unaligned_t *>(scale_row);
        load_step(0, sc0);
        for (int turn = 0; turn < turns; ++turn) {
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's codes of this step are in LDS
            // 16 scales, eight of either step -> word g: blocks 2g, 2g + 1 of the first, then the second
            u32x4 word;
            word[0] = __builtin_amdgcn_perm(sr[2], sr[0], 0x05040100u);
            word[1] = __builtin_amdgcn_perm(sr[2], sr[0], 0x07060302u);
            word[2] = __builtin_amdgcn_perm(sr[3], sr[1], 0x05040100u);
            word[3] = __builtin_amdgcn_perm(sr[3], sr[1], 0x07060302u);
            ss[turn & 1][tid] = word;
            __syncthreads();  // everyone's are, and the other buffer is free
            load_step(2 * turn + 1, sc1);
            sr = *reinterpret_cast<const unaligned_t *>(scale_row + (turn + 1 < turns ? 16 * turn + 16 : 0));
            __builtin_amdgcn_sched_barrier(0);
            const int *sw = reinterpret_cast<const int *>(ss[turn & 1]) + g;
            int as[MT], bs[NT];
#pragma unroll
            for (int t = 0; t < MT; ++t) as[t] = sw[(ar + 16 * t) * 4];
#pragma unroll
            for (int n = 0; n < NT; ++n) bs[n] = sw[(BM + br + item_of<TO>(n, 0)) * 4];
            products(std::integral_constant<int, 0>{}, sc0, as, bs);
            spread(std::integral_constant<int, MT + NT>{});
            __builtin_amdgcn_s_waitcnt(0x0f70);
            __syncthreads();
            load_step(2 * turn + 2, sc0);
            __builtin_amdgcn_sched_barrier(0);
            products(std::integral_constant<int, 1>{}, sc1, as, bs);
            spread(std::integral_constant<int, 0>{});
        }
        __builtin_amdgcn_s_waitcnt(0x0f70);  // (the step loaded for nothing)
    }
#pragma unroll 1
    for (int blk = 16 * turns + g; blk - g < nb; blk += 4) {
        u32x4 af[MT], bf;
        int as[MT], bs;
#pragma unroll
        for (int t = 0; t < MT; ++t)
            load_block(acodes, ascales, a_row(ar + 16 * t), blk, nb, af[t], as[t]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            load_block(codes, scales, b_row(br + item_of<TO>(n, 0)), blk, nb, bf, bs);
#pragma unroll
            for (int t = 0; t < MT; ++t)
                acc[t][n] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                    as_operand(bf), as_operand(af[t]), acc[t][n], 4, 4, 0, bs, 0, as[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int64_t row = row_base + ar + 16 * t;
        TO *dst = out_row<TO>(o, row);
        if (!dst) continue;
        if (rows.of(row) < 0) {
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[t][n] = f32x4{} + __builtin_nanf("");
        }
        put_row<TO, NT>(dst, item_base + wn * NT * 16, g, o.n_items, acc[t]);
    }
}

// ---- launches ------------------------------------------------------------------------------------
template <typename T, typename TO, int NBL, int UT, int NT>
static int launch_narrow(const Rows &rows, const void *a, int width, const uint8_t *codes,
                         const uint8_t *scales, int nb, const ScoreStore &o, hipStream_t st) {
    const int64_t groups = (rows.n_sel + 16 * UT - 1) / (16 * UT);
    const int64_t n_tiles = (o.n_items + 15) / 16;
    // one turn per wave until there are TARGET waves (what the registers let run at once; fewer where
    // eight blocks of activations are split beforehand), then longer walks: 1024, 2048 and 4096
    // waves took 13.8, 14.6 and 11.9 us for 1 x 1000000 x 64 fp32, 18.7, 18.5 and 19.8 for 512 x
    // 26744 x 64, 20.6, 23.6 and 27.8 for 512 x 26744 x 200 bf16, 25.7, 38 and 32 for 1 x 1000000 x
    // 200 fp32
    constexpr int TARGET = NBL == 8 ? 1024 : UT == 1 ? 4096 : 2048;
    int64_t turns = n_tiles * groups / (TARGET * NT);
    turns = turns < 1 ? 1 : (turns > 16 ? 16 : turns);
    const int64_t tpw = turns * NT;
    const int64_t blocks = (n_tiles + 4 * tpw - 1) / (4 * tpw) * groups;
    hipLaunchKernelGGL((mx4_scores_narrow_kernel<T, TO, NBL, UT, NT>), dim3((unsigned)blocks), dim3(256), 0,
                       st, rows, static_cast<const T *>(a), width, codes, scales, nb, o, (int)groups,
                       (int)tpw);
    ALSMI_HIP_CHECK(hipGetLastError());
    return ALSMI_OK;
}

template <typename T, typename TO, int MT, int NT, int KW>
static int launch_wide(const Rows &rows, const void *a, int width, const uint8_t *codes,
                       const uint8_t *scales, int nb, const ScoreStore &o, hipStream_t st) {
    const int64_t groups = (rows.n_sel + 16 * MT - 1) / (16 * MT);
    const int64_t per = 16 * NT * (KW == 1 ? 4 : 1);
    const int64_t blocks = (o.n_items + per - 1) / per * groups;
    hipLaunchKernelGGL((mx4_scores_wide_kernel<T, TO, MT, NT, KW>), dim3((unsigned)blocks), dim3(256), 0,
                       st, rows, static_cast<const T *>(a), width, codes, scales, nb, o, (int)groups);
    ALSMI_HIP_CHECK(hipGetLastError());
    return ALSMI_OK;
}

template <typename TO, int NS, int UT, int NT>
static int launch_both_narrow(const Rows &rows, const void *a, const uint8_t *a_scales,
                              const uint8_t *codes, const uint8_t *scales, int nb, const ScoreStore &o,
                              hipStream_t st) {
    const int64_t groups = (rows.n_sel + 16 * UT - 1) / (16 * UT);
    const int64_t n_tiles = (o.n_items + 15) / 16;
    int64_t turns = n_tiles * groups / (4096 * NT);  // as in launch_narrow
    turns = turns < 1 ? 1 : (turns > 16 ? 16 : turns);
    const int64_t tpw = turns * NT;
    const int64_t blocks = (n_tiles + 4 * tpw - 1) / (4 * tpw) * groups;
    hipLaunchKernelGGL((mx4_scores_both_narrow_kernel<TO, NS, UT, NT>), dim3((unsigned)blocks), dim3(256),
                       0, st, rows, static_cast<const uint8_t *>(a), a_scales, codes, scales, nb, o,
                       (int)groups, (int)tpw);
    ALSMI_HIP_CHECK(hipGetLastError());
    return ALSMI_OK;
}

template <typename TO, int MT, int NT, int KW>
static int launch_both(const Rows &rows, const void *a, const uint8_t *a_scales, const uint8_t *codes,
                       const uint8_t *scales, int nb, const ScoreStore &o, hipStream_t st) {
    const int64_t groups = (rows.n_sel + 16 * MT - 1) / (16 * MT);
    const int64_t per = 16 * NT * (KW == 1 ? 4 : 1);
    const int64_t blocks = (o.n_items + per - 1) / per * groups;
    hipLaunchKernelGGL((mx4_scores_both_kernel<TO, MT, NT, KW>), dim3((unsigned)blocks), dim3(256), 0, st, rows,
                       static_cast<const uint8_t *>(a), a_scales, codes, scales, nb, o, (int)groups);
    ALSMI_HIP_CHECK(hipGetLastError());
    return ALSMI_OK;
}

template <typename TO, int WM, int WN, int MT, int NT>
static int launch_tiled(const Rows &rows, const void *a, const uint8_t *a_scales, const uint8_t *codes,
                        const uint8_t *scales, int nb, const ScoreStore &o, hipStream_t st) {
    constexpr int BM = WM * MT * 16, BN = WN * NT * 16;
    const int64_t row_tiles = (rows.n_sel + BM - 1) / BM;
    const int64_t blocks = (o.n_items + BN - 1) / BN * row_tiles;
    hipLaunchKernelGGL((mx4_scores_tiled_kernel<TO, WM, WN, MT, NT>), dim3((unsigned)blocks),
                       dim3(64 * WM * WN), 0, st, rows, static_cast<const uint8_t *>(a), a_scales, codes,
                       scales, nb, o, (int)row_tiles);
    ALSMI_HIP_CHECK(hipGetLastError());
    return ALSMI_OK;
}

template <typename TO>
static int run_both(const Rows &rows, const void *a, const uint8_t *a_scales, const uint8_t *codes,
                    const uint8_t *scales, int nb, const ScoreStore &o, hipStream_t st) {
    const bool one = rows.n_sel <= 16;
    if (nb <= 4)
        return one ? launch_both_narrow<TO, 1, 1, 2>(rows, a, a_scales, codes, scales, nb, o, st)
                   : launch_both_narrow<TO, 1, 4, 2>(rows, a, a_scales, codes, scales, nb, o, st);
    if (nb <= 8)
        return one ? launch_both_narrow<TO, 2, 1, 2>(rows, a, a_scales, codes, scales, nb, o, st)
                   : launch_both_narrow<TO, 2, 4, 2>(rows, a, a_scales, codes, scales, nb, o, st);
    // (each wave on its own instead of four per row: 1 x 1000000 x 512 72 us instead of 49)
    if (one) return launch_both<TO, 1, 2, 4>(rows, a, a_scales, codes, scales, nb, o, st);
    // the tiled forms keep the loads of a long row in flight, which a few tiles cannot fill the
    // chip with (17 x 4000 x 1024 5.6 us against 4.4, but 40 x 16384 x 4096 15 against 32) and rows of
    // less than a turn have no use for (256 x 4000 x 384 7.3 against 4.6, 128 x 20000 x 300 8.4
    // against 7.2, 1024 x 26744 x 384 in tiles of 128 x 128 33.6 against 32.2)
    const int64_t tiles = (rows.n_sel + 15) / 16 * ((o.n_items + 15) / 16);
    if (tiles < (nb >= 16 ? 2048 : 32768))
        return launch_both<TO, 2, 2, 4>(rows, a, a_scales, codes, scales, nb, o, st);
    // (they load 16 bytes at a time and count a picked row's bytes in 32 bits)
    const bool aligned = (uintptr_t)a % 16 == 0 && (uintptr_t)codes % 16 == 0 &&
                         (!rows.ids || rows.n_rows * nb < (int64_t)1 << 28);
    if (!aligned || nb < 16) return launch_both<TO, 4, 4, 1>(rows, a, a_scales, codes, scales, nb, o, st);
    // A tile of 256 x 256 fills a CU and takes at least 1.1 times less per score than four of 128 x 128,
    // two of which run on a CU at a time; it loses where its last round is not full: 2048 x 16384 x
    // 4096 73 us against 95, 512 x 32768 x 1024 16.8 against 18.4, but 512 x 26744 x 1024 23.5
    // against 19.0, 300 x 65536 x 2048 45 against 41, 1000 x 8192 x 4096 33 against 26.  The blocks
    // behind the last whole turn do not change that (2048 x 16384 x 4000 91 against 131, x 992 44
    // against 52 and 68 from memory), though read from memory they take their time: x 4096 takes
    // 73 us, x 2000 59 (x 2048 44), x 1024 31.
    const int64_t t256 = (rows.n_sel + 255) / 256 * ((o.n_items + 255) / 256);
    const int64_t t128 = (rows.n_sel + 127) / 128 * ((o.n_items + 127) / 128);
    if ((t256 + 255) / 256 * 102400 <= t128 * 115)
        return launch_tiled<TO, 4, 2, 4, 8>(rows, a, a_scales, codes, scales, nb, o, st);
    return launch_tiled<TO, 2, 2, 4, 4>(rows, a, a_scales, codes, scales, nb, o, st);
}

// Whether a float product is split first: enough whole tiles (bf16, 128 x 16384 x 512 11.8 us against
// 15.8 from memory, 512 x 4096 x 1024 18.9 against 27.6, but 128 x 8192 x 4096 53 against 48), for up
// to 64 rows, which leave half of a tile empty, only long rows and more tiles (64 x 65536 x 2048 fp32
// 87 against 133, 64 x 100000 x 512 fp32 49 against 45, 64 x 16384 x 4096 bf16 53 against 47).
static bool splits(int64_t n_sel, int64_t n_items, int nb) {
    const int64_t tiles = (n_sel + WT_ROWS - 1) / WT_ROWS * ((n_items + WT_ITEMS - 1) / WT_ITEMS);
    return n_sel > 64 ? nb > 8 && tiles >= 128 : n_sel > 32 && nb >= 32 && tiles >= 192;
}
static int64_t split_bytes(int64_t n_sel, int nb, int parts) {
    return n_sel * ((nb + 3) / 4) * 256 * parts;
}
static int parts_of(int dtype) {
    return dtype == ALSMI_F32 ? 3 : dtype == ALSMI_F16 ? 2 : dtype == ALSMI_BF16 ? 1 : 0;
}
// Rows and items that a product takes at once, so that a launch has fewer than 2^32 threads: where the
// waves of a workgroup share rows it covers no more than 32 items (and then up to 32 rows, or fewer
// than 32768 tiles, are left).  Rows that are split first: whole tiles whose parts take 256 MiB.
constexpr int64_t MX4_ITEMS = (int64_t)1 << 28;
static int64_t batch_rows(int dtype, int64_t n_sel, int64_t n_items, int nb) {
    if (dtype == ALSMI_MX4 || !splits(n_sel, n_items, nb)) return (int64_t)1 << 22;
    const int64_t fit = MX4_SPLIT_BYTES / split_bytes(1, nb, parts_of(dtype));
    return std::max<int64_t>(WT_ROWS, fit / WT_ROWS * WT_ROWS);
}

template <typename T, typename TO, int WN>
static int launch_split(const Rows &rows, const void *a, int width, const uint8_t *codes,
                        const uint8_t *scales, int nb, const ScoreStore &o, void *workspace,
                        hipStream_t st) {
    u32x4 *planes = static_cast<u32x4 *>(workspace);
    const int64_t row_tiles = (rows.n_sel + WT_ROWS - 1) / WT_ROWS;
    const int64_t blocks = (o.n_items + 64 * WN - 1) / (64 * WN) * row_tiles;
    hipLaunchKernelGGL((mx4_split_kernel<T>), dim3((unsigned)rows.n_sel), dim3(256), 0, st, rows,
                       static_cast<const T *>(a), width, (nb + 3) / 4 * 16, planes);
    ALSMI_HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL((mx4_scores_split_kernel<TO, Parts<T>::N, WN>), dim3((unsigned)blocks),
                       dim3(128 * WN), 0, st, planes, codes, scales, nb, o, (int)row_tiles);
    ALSMI_HIP_CHECK(hipGetLastError());
    return ALSMI_OK;
}

template <typename T, typename TO>
static int run_scores(const Rows &rows, const void *a, int width, const uint8_t *codes,
                      const uint8_t *scales, int nb, const ScoreStore &o, bool split, void *workspace,
                      hipStream_t st) {
    if (split) {
        // 256 items a workgroup read each part half as often, which pays for three parts and enough
        // tiles (65 x 40000 x 512 fp32 24.6 us against 33.4, 2048 x 16384 x 4096 629 against 819, but 128 x
        // 16384 x 512 25.6 against 19.8; fp16 2000 x 16000 x 2000 257 against 262, bf16 171 against 156)
        if constexpr (Parts<T>::N > 2) {
            if ((rows.n_sel + WT_ROWS - 1) / WT_ROWS * ((o.n_items + 255) / 256) >= 128)
                return launch_split<T, TO, 4>(rows, a, width, codes, scales, nb, o, workspace, st);
        }
        return launch_split<T, TO, 2>(rows, a, width, codes, scales, nb, o, workspace, st);
    }
    const bool one = rows.n_sel <= 16;
    if (nb == 1)
        return one ? launch_narrow<T, TO, 1, 1, 2>(rows, a, width, codes, scales, nb, o, st)
                   : launch_narrow<T, TO, 1, 4, 2>(rows, a, width, codes, scales, nb, o, st);
    if (nb == 2)
        return one ? launch_narrow<T, TO, 2, 1, 2>(rows, a, width, codes, scales, nb, o, st)
                   : launch_narrow<T, TO, 2, 4, 2>(rows, a, width, codes, scales, nb, o, st);
    // (three parts of four tiles at four blocks would need 192 registers)
    if (nb <= 4)
        return one ? launch_narrow<T, TO, 4, 1, 2>(rows, a, width, codes, scales, nb, o, st)
                   : launch_narrow<T, TO, 4, 2, 2>(rows, a, width, codes, scales, nb, o, st);
    // (eight blocks in the forms below: 1 x 500000 x 200 fp32 40 us instead of 21, 1024 x 32000 x 200
    // fp32 87 instead of 59, bf16 39 instead of 36)
    if (nb <= 8)
        return one ? launch_narrow<T, TO, 8, 1, 2>(rows, a, width, codes, scales, nb, o, st)
                   : launch_narrow<T, TO, 8, 4 / Parts<T>::N, 2>(rows, a, width, codes, scales, nb, o, st);
    // Four waves share a row's contraction, or each forms tiles of its own and reads the activations
    // less often, which pays for several parts and many items against short rows: 1 x 1000000 x 512
    // fp32 105 us against 84, 16 x 400000 x 1024 141 against 109, but 1 x 100000 x 4096 80 against
    // 121; bf16 1 x 400000 x 1024 70 against 85, 16 x 1000000 x 512 120 against 108.
    const int64_t tiles = (rows.n_sel + 15) / 16 * ((o.n_items + 15) / 16);
    const int steps = (nb + 3) / 4;
    if (one)
        return Parts<T>::N == 1 || tiles < 2048 * (int64_t)steps
                   ? launch_wide<T, TO, 1, 2, 4>(rows, a, width, codes, scales, nb, o, st)
                   : launch_wide<T, TO, 1, 4, 1>(rows, a, width, codes, scales, nb, o, st);
    // two row tiles a wave, or four: 17 x 200000 x 1024 bf16 59 us against 81, 64 x 16384 x 2000 fp32
    // 39 against 110, but 64 x 65536 x 512 45 against 37, 33 x 100000 x 512 60 against 39
    return rows.n_sel <= 32 || tiles < 16384
               ? launch_wide<T, TO, 2, 2, 4>(rows, a, width, codes, scales, nb, o, st)
               : launch_wide<T, TO, 4, 4, 1>(rows, a, width, codes, scales, nb, o, st);
}

}  // namespace alsmi

extern "C" {

int alsmi_mx4_quantize(int dtype, int64_t n_rows, int64_t width, const void *x, int64_t ldx,
                       uint8_t *codes, uint8_t *scales, void *stream) {
    using namespace alsmi;
    ALSMI_REQUIRE(dtype >= ALSMI_F32 && dtype <= ALSMI_BF16, "alsmi_mx4_quantize: bad dtype %d", dtype);
    ALSMI_REQUIRE(n_rows >= 0 && n_rows <= INT32_MAX, "alsmi_mx4_quantize: bad row count %lld",
                  (long long)n_rows);
    ALSMI_REQUIRE(width >= 1 && width <= MX4_MAX_WIDTH, "alsmi_mx4_quantize: width %lld outside 1..%lld",
                  (long long)width, (long long)MX4_MAX_WIDTH);
    if (n_rows == 0) return ALSMI_OK;
    ALSMI_REQUIRE(ldx >= width || n_rows == 1, "alsmi_mx4_quantize: row stride %lld below the width",
                  (long long)ldx);
    ALSMI_REQUIRE(x && codes && scales, "alsmi_mx4_quantize: null pointer");
    ALSMI_REQUIRE((uintptr_t)codes % 4 == 0, "alsmi_mx4_quantize: codes must be aligned to 4 bytes");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int nb = (int)((width + MX4_BLOCK - 1) / MX4_BLOCK);
#define ALSMI_CASE(T)                                                                                \
    do {                                                                                             \
        const RowGrid rg = row_grid(nb, mx4_lane<T>());                                              \
        auto kernel = n_rows * width * (int64_t)sizeof(T) > MX4_STREAM_BYTES                         \
                          ? mx4_quantize_kernel<T, true>                                             \
                          : mx4_quantize_kernel<T, false>;                                           \
        for (int64_t lo = 0; lo < n_rows; lo += rg.most) {                                           \
            const int64_t n = std::min(n_rows - lo, rg.most);                                        \
            hipLaunchKernelGGL(kernel, rg.grid(n), dim3(256), 0, st, n, (int)width,                  \
                               static_cast<const T *>(x) + lo * ldx, ldx, codes + lo * nb * 16,      \
                               scales + lo * nb, rg.upr, rg.rpb, rg.inverse);                        \
            ALSMI_HIP_CHECK(hipGetLastError());                                                      \
        }                                                                                            \
    } while (0)
    if (dtype == ALSMI_F32) ALSMI_CASE(float);
    else if (dtype == ALSMI_F64) ALSMI_CASE(double);
    else if (dtype == ALSMI_F16) ALSMI_CASE(_Float16);
    else ALSMI_CASE(__bf16);
#undef ALSMI_CASE
    return ALSMI_OK;
}

int alsmi_mx4_dequantize(int dtype, int64_t n_sel, const int32_t *rows, int64_t n_rows, int64_t width,
                         const uint8_t *codes, const uint8_t *scales, void *out, int64_t ldo,
                         void *stream) {
    using namespace alsmi;
    ALSMI_REQUIRE(dtype >= ALSMI_F32 && dtype <= ALSMI_BF16, "alsmi_mx4_dequantize: bad dtype %d",
                  dtype);
    ALSMI_REQUIRE(n_rows >= 0 && n_rows <= INT32_MAX && n_sel >= 0 && n_sel <= INT32_MAX,
                  "alsmi_mx4_dequantize: bad row count");
    ALSMI_REQUIRE(rows || n_sel <= n_rows, "alsmi_mx4_dequantize: %lld rows of a table of %lld",
                  (long long)n_sel, (long long)n_rows);
    ALSMI_REQUIRE(width >= 1 && width <= MX4_MAX_WIDTH,
                  "alsmi_mx4_dequantize: width %lld outside 1..%lld", (long long)width,
                  (long long)MX4_MAX_WIDTH);
    if (n_sel == 0) return ALSMI_OK;
    ALSMI_REQUIRE(ldo >= width || n_sel == 1, "alsmi_mx4_dequantize: row stride %lld below the width",
                  (long long)ldo);
    ALSMI_REQUIRE(out && (n_rows == 0 || (codes && scales)), "alsmi_mx4_dequantize: null pointer");
    ALSMI_REQUIRE((uintptr_t)codes % 4 == 0, "alsmi_mx4_dequantize: codes must be aligned to 4 bytes");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int nb = (int)((width + MX4_BLOCK - 1) / MX4_BLOCK);
#define ALSMI_CASE(T)                                                                                 \
    do {                                                                                              \
        const RowGrid rg = row_grid(nb, mx4_lane<T>());                                               \
        auto kernel = n_sel * width * (int64_t)sizeof(T) > MX4_STREAM_BYTES                           \
                          ? mx4_dequantize_kernel<T, true>                                            \
                          : mx4_dequantize_kernel<T, false>;                                          \
        for (int64_t lo = 0; lo < n_sel; lo += rg.most) {                                             \
            const int64_t n = std::min(n_sel - lo, rg.most), skip = rows ? 0 : lo;                    \
            hipLaunchKernelGGL(kernel, rg.grid(n), dim3(256), 0, st, n, rows ? rows + lo : nullptr,   \
                               n_rows - skip, (int)width, codes + skip * nb * 16, scales + skip * nb, \
                               static_cast<T *>(out) + lo * ldo, ldo, rg.upr, rg.rpb, rg.inverse);    \
            ALSMI_HIP_CHECK(hipGetLastError());                                                       \
        }                                                                                             \
    } while (0)
    if (dtype == ALSMI_F32) ALSMI_CASE(float);
    else if (dtype == ALSMI_F64) ALSMI_CASE(double);
    else if (dtype == ALSMI_F16) ALSMI_CASE(_Float16);
    else ALSMI_CASE(__bf16);
#undef ALSMI_CASE
    return ALSMI_OK;
}

size_t alsmi_mx4_scores_workspace_bytes(int dtype, int64_t n_sel, int64_t n_items, int64_t width) {
    using namespace alsmi;
    if (n_sel < 0 || n_items < 0 || width < 1 || width > MX4_MAX_WIDTH) return 0;
    const int nb = (int)((width + MX4_BLOCK - 1) / MX4_BLOCK);
    if (!splits(n_sel, n_items, nb)) return 0;
    // (enough for fewer rows or items or a smaller width as well)
    const int64_t all = split_bytes(n_sel, nb, parts_of(dtype)), least = split_bytes(WT_ROWS, nb, parts_of(dtype));
    return (size_t)std::min(all, std::max(MX4_SPLIT_BYTES, least));
}

int alsmi_mx4_scores(int dtype, int64_t n_sel, const int32_t *rows, int64_t n_rows, const void *a,
                     int64_t lda, const uint8_t *a_scales, int64_t n_items, int64_t width,
                     const uint8_t *codes, const uint8_t *scales, int out_dtype, void *out,
                     int64_t ldo, void *workspace, void *stream) {
    using namespace alsmi;
    ALSMI_REQUIRE(dtype == ALSMI_F32 || dtype == ALSMI_F16 || dtype == ALSMI_BF16 || dtype == ALSMI_MX4,
                  "alsmi_mx4_scores: bad dtype %d", dtype);
    ALSMI_REQUIRE(out_dtype == ALSMI_F32 || out_dtype == ALSMI_F16 || out_dtype == ALSMI_BF16,
                  "alsmi_mx4_scores: bad output dtype %d", out_dtype);
    ALSMI_REQUIRE(n_rows >= 0 && n_rows <= INT32_MAX && n_sel >= 0 && n_sel <= INT32_MAX &&
                      n_items >= 0 && n_items <= INT32_MAX,
                  "alsmi_mx4_scores: bad row or item count");
    ALSMI_REQUIRE(rows || n_sel <= n_rows, "alsmi_mx4_scores: %lld rows of a table of %lld",
                  (long long)n_sel, (long long)n_rows);
    ALSMI_REQUIRE(width >= 1 && width <= MX4_MAX_WIDTH, "alsmi_mx4_scores: width %lld outside 1..%lld",
                  (long long)width, (long long)MX4_MAX_WIDTH);
    if (n_sel == 0 || n_items == 0) return ALSMI_OK;
    ALSMI_REQUIRE(n_rows > 0, "alsmi_mx4_scores: rows of an empty table");
    ALSMI_REQUIRE(ldo >= n_items || n_sel == 1, "alsmi_mx4_scores: output stride %lld below n_items",
                  (long long)ldo);
    ALSMI_REQUIRE(dtype == ALSMI_MX4 || lda >= width || n_rows == 1,
                  "alsmi_mx4_scores: row stride %lld below the width", (long long)lda);
    ALSMI_REQUIRE(a && codes && scales && out && (dtype != ALSMI_MX4 || a_scales),
                  "alsmi_mx4_scores: null pointer");
    ALSMI_REQUIRE((uintptr_t)codes % 4 == 0 && (dtype != ALSMI_MX4 || (uintptr_t)a % 4 == 0),
                  "alsmi_mx4_scores: codes must be aligned to 4 bytes");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int nb = (int)((width + MX4_BLOCK - 1) / MX4_BLOCK);
    ALSMI_REQUIRE(alsmi_mx4_scores_workspace_bytes(dtype, n_sel, n_items, width) == 0 ||
                      (workspace && (uintptr_t)workspace % 16 == 0),
                  "alsmi_mx4_scores: needs a workspace aligned to 16 bytes");
    const bool split = splits(n_sel, n_items, nb) && (uintptr_t)codes % 16 == 0;
    const int64_t most = batch_rows(dtype, n_sel, n_items, nb);
    const int64_t out_size = out_dtype == ALSMI_F32 ? 4 : 2;
    // bytes of a row of the activations
    const int64_t a_row = dtype == ALSMI_MX4 ? 16 * nb : lda * (dtype == ALSMI_F32 ? 4 : 2);
    auto product = [&](int64_t lo, int64_t first) {
        const int64_t n = std::min(n_sel - lo, most), skip = rows ? 0 : lo;
        const Rows r = {n, n_rows - skip, lda, rows ? rows + lo : nullptr};
        const ScoreStore o = {static_cast<char *>(out) + (lo * ldo + first) * out_size, ldo, n,
                              std::min(n_items - first, MX4_ITEMS)};
        const void *from = static_cast<const char *>(a) + skip * a_row;
        const uint8_t *from_scales = a_scales ? a_scales + skip * nb : nullptr;
        const uint8_t *c = codes + first * nb * 16, *sc = scales + first * nb;
#define ALSMI_CASE(TO)                                                                                  \
    do {                                                                                                \
        if (dtype == ALSMI_F32)                                                                         \
            return run_scores<float, TO>(r, from, (int)width, c, sc, nb, o, split, workspace, st);      \
        if (dtype == ALSMI_F16)                                                                         \
            return run_scores<_Float16, TO>(r, from, (int)width, c, sc, nb, o, split, workspace, st);   \
        if (dtype == ALSMI_BF16)                                                                        \
            return run_scores<__bf16, TO>(r, from, (int)width, c, sc, nb, o, split, workspace, st);     \
        return run_both<TO>(r, from, from_scales, c, sc, nb, o, st);                                    \
    } while (0)
        if (out_dtype == ALSMI_F32) ALSMI_CASE(float);
        if (out_dtype == ALSMI_BF16) ALSMI_CASE(__bf16);
        ALSMI_CASE(_Float16);
#undef ALSMI_CASE
    };
    for (int64_t lo = 0; lo < n_sel; lo += most)
        for (int64_t first = 0; first < n_items; first += MX4_ITEMS) {
            const int status = product(lo, first);
            if (status != ALSMI_OK) return status;
        }
    return ALSMI_OK;
}

}  // extern "C"
