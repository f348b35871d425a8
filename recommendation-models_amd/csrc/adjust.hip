// Score rows changed by what is known of the row before the selection: penalties for the items of a
// history (or their exclusion), biases, availability masks.
//
// Per row r and item i, c = occurrences of i in the row's history:
//   c > 0:  x = s > 0 ? s / repetition : s * repetition, then x -= frequency * c + presence;
//   c == 0: x = s
//   x += item_bias[i];  x += the value of the LAST entry of i in the row's bias list
//   x = -inf where the row's mask has no bit i, or (exclude) c > 0
// One pass over the scores.  The sparse lists of a row are turned into bits and counters in LDS for the
// tile of items a workgroup owns: a scan of the list, integer atomics (their order cannot change
// the result), no sorting and no second launch.  Bound by the read and the write of the scores
// (1024 x 26744 fp32 with exclusion, bias and masks: 47 us, 4.7 TB/s, or 35 us for scores that the
// call before left in the last-level cache), for long lists over many tiles by latencies: first
// the lists, behind the barrier mask, penalties and biases (64 x 131072 bf16, lists of 900 on
// average: 13.6 us; 61 % of the waves' cycles are waits, the vector instructions fill a third of
// the time).
#include "alsmi_common.h"
#include "elem.h"

#include <algorithm>
#include <type_traits>

namespace alsmi {

constexpr int ADJ_THREADS = 256;
constexpr unsigned ADJ_TILE = ADJ_THREADS * 8;  // items of a workgroup

// Entries [lo, hi) of row `row` of a ragged list, inside the list whatever the pointers hold.
__device__ __forceinline__ void list_range(const int64_t *ptr, int64_t row, int64_t n, int64_t &lo,
                                           int64_t &hi) {
    lo = ptr[row];
    hi = ptr[row + 1];
    lo = lo < 0 ? 0 : (lo > n ? n : lo);
    hi = hi < lo ? lo : (hi > n ? n : hi);
}

// Entries [lo, hi) of a ragged list whose ids fall into the workgroup's tile: f(index in the tile, entry
// counted from lo).  Four loads in flight per thread.  (An id outside the items, such as a pad
// entry of -1, falls into no tile: the last one is cut at n_items.)
template <typename F>
__device__ __forceinline__ void scan_list(const int32_t *__restrict__ ids, int64_t lo, int64_t hi,
                                          unsigned first, unsigned in_tile, F f) {
    const int32_t *list = ids + lo;
    const unsigned n = (unsigned)(hi - lo);
    for (unsigned e = threadIdx.x; e < n; e += 4 * ADJ_THREADS) {
        unsigned at[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const unsigned k = e + u * ADJ_THREADS;
            at[u] = (unsigned)list[k < n ? k : e] - first;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (e + u * ADJ_THREADS < n && at[u] < in_tile) f(at[u], e + u * ADJ_THREADS);
    }
}

// x where bit i of `bits` is set, else -inf
__device__ __forceinline__ float keep(float x, unsigned bits, int i) {
    const unsigned all = (unsigned)__builtin_amdgcn_sbfe((int)bits, i, 1);
    return __builtin_bit_cast(float, (__builtin_bit_cast(unsigned, x) & all) | (0xff800000u & ~all));
}
__device__ __forceinline__ double keep(double x, unsigned bits, int i) {
    return (bits >> i) & 1u ? x : -__builtin_inf();
}

// A workgroup owns ADJ_TILE items of a row, eight consecutive ones per thread, whose scores are on their
// way while the lists are read (tiles of 4096 and 8192 took 4 % and 40 % longer at 1024 x 26744).
// In LDS one bit per item says that a list holds it (all that an exclusion needs: it joins the mask),
// one word per item and list how often, or by which entry: only threads with a bit set look at the
// words (looking at all of them cost 42 us instead of 37 there).
template <typename T>
__global__ __launch_bounds__(ADJ_THREADS) void adjust_kernel(alsmi_adjust a, const T *scores, T *out,
                                                             unsigned tiles, unsigned first_row) {
    typedef typename Elem<T>::wide W;
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    __shared__ unsigned seen[ADJ_TILE / 32], biased[ADJ_TILE / 32];
    __shared__ u32x4 count4[ADJ_TILE / 4], last4[ADJ_TILE / 4];
    unsigned *count = reinterpret_cast<unsigned *>(count4), *last = reinterpret_cast<unsigned *>(last4);
    const unsigned tid = threadIdx.x;
    const unsigned r32 = blockIdx.x / tiles;
    const int64_t row = (int64_t)first_row + r32;
    const unsigned first = (blockIdx.x - r32 * tiles) * ADJ_TILE;
    const unsigned n_items = (unsigned)a.n_items;
    const unsigned in_tile = n_items - first < ADJ_TILE ? n_items - first : ADJ_TILE;
    const T *src = scores + row * a.ld_scores + first;
    T *dst = out + row * a.ld_out + first;
    const unsigned at = tid * 8;
    W x[8];
    load8<T>(x, src + at, (int)(in_tile - at));
    int64_t h0 = 0, h1 = 0, b0 = 0, b1 = 0;
    if (a.history_ptr) {
        const int64_t hr = a.history_rows ? (int64_t)a.history_rows[row] : row;
        if (hr >= 0 && hr < a.n_history_rows) list_range(a.history_ptr, hr, a.n_history, h0, h1);
    }
    if (a.bias_ptr) list_range(a.bias_ptr, row, a.n_bias, b0, b1);
    const bool has_h = h1 > h0, has_b = b1 > b0;  // (the same for the whole workgroup)
    const uint8_t *mask = nullptr;
    bool none = false;
    if (a.mask) {
        const int64_t mr = a.mask_rows ? (int64_t)a.mask_rows[row] : (a.n_masks == 1 ? 0 : row);
        if (mr >= a.n_masks) none = true;
        else if (mr >= 0)
            mask = reinterpret_cast<const uint8_t *>(a.mask + mr * ((a.n_items + 31) / 32)) + first / 8;
    }
    if (has_h || has_b) {
        for (unsigned i = tid; i < ADJ_TILE / 32; i += ADJ_THREADS) seen[i] = biased[i] = 0;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            if (has_h && !a.exclude) count4[v * ADJ_THREADS + tid] = u32x4{0, 0, 0, 0};
            if (has_b) last4[v * ADJ_THREADS + tid] = u32x4{0, 0, 0, 0};
        }
        __syncthreads();
        if (has_h) {
            if (a.exclude)
                scan_list(a.history_ids, h0, h1, first, in_tile,
                          [&](unsigned i, unsigned) { atomicOr(&seen[i >> 5], 1u << (i & 31)); });
            else
                scan_list(a.history_ids, h0, h1, first, in_tile, [&](unsigned i, unsigned) {
                    atomicOr(&seen[i >> 5], 1u << (i & 31));
                    atomicAdd(&count[i], 1u);
                });
        }
        if (has_b)
            scan_list(a.bias_ids, b0, b1, first, in_tile, [&](unsigned i, unsigned e) {
                atomicOr(&biased[i >> 5], 1u << (i & 31));
                atomicMax(&last[i], e + 1u);
            });
        __syncthreads();
    }
    if (at >= in_tile) return;
    unsigned allowed = none ? 0u : 0xffu;
    if (mask) allowed = mask[at >> 3];
    if (has_h) {
        const unsigned hits = reinterpret_cast<const uint8_t *>(seen)[at >> 3];
        if (a.exclude) {
            allowed &= ~hits;
        } else if (hits) {
            W rep = (W)a.repetition_value, freq = (W)a.frequency_value, pres = (W)a.presence_value;
            if (a.repetition) rep = (W)a.repetition[row];
            if (a.frequency) freq = (W)a.frequency[row];
            if (a.presence) pres = (W)a.presence[row];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if ((hits >> i) & 1u) {
                    const W s = x[i];
                    x[i] = (s > 0 ? s / rep : s * rep) - (freq * (W)count[at + i] + pres);
                }
        }
    }
    if (a.item_bias) {
        auto add = [&](const auto *bias) {
            typename std::remove_const<typename std::remove_pointer<decltype(bias)>::type>::type b[8];
            load8(b, bias + first + at, (int)(in_tile - at));
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] += (W)b[i];
        };
        if (sizeof(T) == 8 && a.item_bias_dtype == ALSMI_F64) add(static_cast<const double *>(a.item_bias));
        else add(static_cast<const float *>(a.item_bias));
    }
    if (has_b) {
        const unsigned hits = reinterpret_cast<const uint8_t *>(biased)[at >> 3];
        if (hits) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if ((hits >> i) & 1u) x[i] += (W)a.bias_values[b0 + (int64_t)(last[at + i] - 1u)];
        }
    }
    if (allowed != 0xffu) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = keep(x[i], allowed, i);
    }
    store8<T>(dst + at, x, (int)(in_tile - at));
}

template <typename T>
static int run_adjust(const alsmi_adjust &a, const void *scores, void *out, hipStream_t st) {
    const int64_t tiles = (a.n_items + ADJ_TILE - 1) / ADJ_TILE;
    const int64_t most = std::max<int64_t>(1, ((int64_t)1 << 23) / tiles);  // (under 2^32 threads a launch)
    for (int64_t lo = 0; lo < a.n_rows; lo += most) {
        const int64_t rows = std::min(a.n_rows - lo, most);
        hipLaunchKernelGGL((adjust_kernel<T>), dim3((unsigned)(tiles * rows)), dim3(ADJ_THREADS), 0, st, a,
                           static_cast<const T *>(scores), static_cast<T *>(out), (unsigned)tiles,
                           (unsigned)lo);
        ALSMI_HIP_CHECK(hipGetLastError());
    }
    return ALSMI_OK;
}

}  // namespace alsmi

extern "C" int alsmi_adjust_scores(int dtype, const alsmi_adjust *args, const void *scores, void *out,
                                   void *stream) {
    using namespace alsmi;
    ALSMI_REQUIRE(dtype >= ALSMI_F32 && dtype <= ALSMI_BF16, "alsmi_adjust_scores: bad dtype %d", dtype);
    ALSMI_REQUIRE(args, "alsmi_adjust_scores: null pointer");
    const alsmi_adjust a = *args;
    ALSMI_REQUIRE(a.n_rows >= 0 && a.n_rows <= INT32_MAX && a.n_items >= 0 && a.n_items <= INT32_MAX,
                  "alsmi_adjust_scores: bad row or item count");
    if (a.n_rows == 0 || a.n_items == 0) return ALSMI_OK;
    ALSMI_REQUIRE((a.ld_scores >= a.n_items && a.ld_out >= a.n_items) || a.n_rows == 1,
                  "alsmi_adjust_scores: row stride below n_items");
    ALSMI_REQUIRE(scores && out, "alsmi_adjust_scores: null pointer");
    ALSMI_REQUIRE(!a.history_ptr || (a.n_history >= 0 && a.n_history <= INT32_MAX &&
                                     (a.n_history == 0 || a.history_ids) &&
                                     (a.history_rows ? a.n_history_rows >= 0
                                                     : a.n_history_rows >= a.n_rows)),
                  "alsmi_adjust_scores: history lists do not fit the rows");
    ALSMI_REQUIRE(!a.bias_ptr || (a.n_bias >= 0 && a.n_bias <= INT32_MAX &&
                                  (a.n_bias == 0 || (a.bias_ids && a.bias_values))),
                  "alsmi_adjust_scores: bias lists without ids or values");
    ALSMI_REQUIRE(!a.item_bias || a.item_bias_dtype == ALSMI_F32 ||
                      (a.item_bias_dtype == ALSMI_F64 && dtype == ALSMI_F64),
                  "alsmi_adjust_scores: bad item bias dtype %d", a.item_bias_dtype);
    ALSMI_REQUIRE(!a.mask || (a.mask_rows ? a.n_masks >= 0 : a.n_masks == 1 || a.n_masks >= a.n_rows),
                  "alsmi_adjust_scores: fewer masks than rows");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == ALSMI_F32) return run_adjust<float>(a, scores, out, st);
    if (dtype == ALSMI_F64) return run_adjust<double>(a, scores, out, st);
    if (dtype == ALSMI_F16) return run_adjust<_Float16>(a, scores, out, st);
    return run_adjust<__bf16>(a, scores, out, st);
}
