// Score rows changed by what is known of the row before the selection: penalties for the items of a
// history (or their exclusion), biases, availability masks.
//
// Per row r and item i, c = occurrences of i in the row's history:
//   c > 0:  x = -inf (exclude), else x = s > 0 ? s / repetition : s * repetition, then
//           x -= frequency * c + presence;      otherwise x = s
//   x += item_bias[i];  x += the value of the LAST entry of i in the row's bias list
//   x = -inf where the row's mask has no bit i
// One pass over the scores.  The sparse lists of a row are turned into dense counters in LDS for the
// tile of items a workgroup owns: a scan of the list, integer atomics (their order cannot change
// the result), no sorting and no second launch.  Bound by the read and the write of the scores.
#include "alsmi_common.h"
#include "elem.h"

namespace alsmi {

constexpr int ADJ_THREADS = 256;
constexpr int ADJ_STEP = ADJ_THREADS * 8;  // items a workgroup takes per turn, eight per thread

// Entries [lo, hi) of row `row` of a ragged list, inside the list whatever the pointers hold.
__device__ __forceinline__ void list_range(const int64_t *ptr, int64_t row, int64_t n, int64_t &lo,
                                           int64_t &hi) {
    lo = ptr[row];
    hi = ptr[row + 1];
    lo = lo < 0 ? 0 : (lo > n ? n : lo);
    hi = hi < lo ? lo : (hi > n ? n : hi);
}

template <typename T, int V>
__global__ __launch_bounds__(ADJ_THREADS) void adjust_kernel(alsmi_adjust a, const T *scores, T *out,
                                                             unsigned tiles) {
    typedef typename Elem<T>::wide W;
    constexpr int TILE = ADJ_STEP * V;
    __shared__ unsigned count[TILE];
    __shared__ unsigned last[TILE];
    const int tid = threadIdx.x;
    const unsigned r32 = blockIdx.x / tiles;
    const int64_t row = r32;
    const int64_t first = (int64_t)(blockIdx.x - r32 * tiles) * TILE;
    const T *src = scores + row * a.ld_scores;
    T *dst = out + row * a.ld_out;
    // the scores are on their way while the lists are read
    W x[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int64_t at = first + v * ADJ_STEP + tid * 8;
        load8<T>(x[v], src + at, a.n_items - at);
    }
    int64_t h0 = 0, h1 = 0, b0 = 0, b1 = 0;
    if (a.history_ptr) {
        const int64_t hr = a.history_rows ? (int64_t)a.history_rows[row] : row;
        if (hr >= 0 && hr < a.n_history_rows) list_range(a.history_ptr, hr, a.n_history, h0, h1);
    }
    if (a.bias_ptr) list_range(a.bias_ptr, row, a.n_bias, b0, b1);
    const bool has_h = h1 > h0, has_b = b1 > b0;  // (the same for the whole workgroup)
    if (has_h || has_b) {
        for (int i = tid; i < TILE; i += ADJ_THREADS) {
            if (has_h) count[i] = 0;
            if (has_b) last[i] = 0;
        }
        __syncthreads();
        // (an id outside the items, such as a pad entry of -1, lies in no tile)
        for (int64_t e = h0 + tid; e < h1; e += ADJ_THREADS) {
            const int64_t i = (int64_t)a.history_ids[e] - first;
            if (i >= 0 && i < TILE) atomicAdd(&count[i], 1u);
        }
        for (int64_t e = b0 + tid; e < b1; e += ADJ_THREADS) {
            const int64_t i = (int64_t)a.bias_ids[e] - first;
            if (i >= 0 && i < TILE) atomicMax(&last[i], (unsigned)(e - b0) + 1u);
        }
        __syncthreads();
    }
    W rep = (W)a.repetition_value, freq = (W)a.frequency_value, pres = (W)a.presence_value;
    if (a.repetition) rep = (W)a.repetition[row];
    if (a.frequency) freq = (W)a.frequency[row];
    if (a.presence) pres = (W)a.presence[row];
    const uint8_t *mask = nullptr;
    bool none = false;
    if (a.mask) {
        const int64_t mr = a.mask_rows ? (int64_t)a.mask_rows[row] : (a.n_masks == 1 ? 0 : row);
        if (mr >= a.n_masks) none = true;
        else if (mr >= 0)
            mask = reinterpret_cast<const uint8_t *>(a.mask) + mr * ((a.n_items + 31) / 32) * 4;
    }
    const W neg_inf = -(W)__builtin_inf();
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int local = v * ADJ_STEP + tid * 8;
        const int64_t at = first + local;
        if (at >= a.n_items) continue;
        if (has_h) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned c = count[local + i];
                if (c == 0) continue;
                if (a.exclude) {
                    x[v][i] = neg_inf;
                } else {
                    const W s = x[v][i];
                    x[v][i] = (s > 0 ? s / rep : s * rep) - (freq * (W)c + pres);
                }
            }
        }
        if (a.item_bias) {
            float b[8];
            load8<float>(b, a.item_bias + at, a.n_items - at);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[v][i] += (W)b[i];
        }
        if (has_b) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned e = last[local + i];
                if (e) x[v][i] += (W)a.bias_values[b0 + (int64_t)(e - 1u)];
            }
        }
        if (mask || none) {
            const unsigned bits = none ? 0u : mask[at >> 3];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[v][i] = (bits >> i) & 1u ? x[v][i] : neg_inf;
        }
        store8<T>(dst + at, x[v], a.n_items - at);
    }
}

template <typename T>
static int run_adjust(const alsmi_adjust &a, const void *scores, void *out, hipStream_t st) {
    const int64_t tiles = (a.n_items + ADJ_STEP - 1) / ADJ_STEP;
    ALSMI_REQUIRE(tiles * a.n_rows <= INT32_MAX, "alsmi_adjust_scores: too many rows x items");
    hipLaunchKernelGGL((adjust_kernel<T, 1>), dim3((unsigned)(tiles * a.n_rows)), dim3(ADJ_THREADS), 0,
                       st, a, static_cast<const T *>(scores), static_cast<T *>(out), (unsigned)tiles);
    ALSMI_HIP_CHECK(hipGetLastError());
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
    ALSMI_REQUIRE(!a.mask || (a.mask_rows ? a.n_masks >= 0 : a.n_masks == 1 || a.n_masks >= a.n_rows),
                  "alsmi_adjust_scores: fewer masks than rows");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == ALSMI_F32) return run_adjust<float>(a, scores, out, st);
    if (dtype == ALSMI_F64) return run_adjust<double>(a, scores, out, st);
    if (dtype == ALSMI_F16) return run_adjust<_Float16>(a, scores, out, st);
    return run_adjust<__bf16>(a, scores, out, st);
}
