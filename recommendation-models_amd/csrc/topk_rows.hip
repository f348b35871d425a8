// The k largest scores of every row of a score block, best first, ties to the lowest index.
//
// Scores are ranked through the order-preserving integer image of their bits joined with the
// complement of their index: (image << 32) | ~index.  These keys are all different, so "the k-th
// largest" is one element however many scores are equal (rows that a mask left mostly at -inf, 16-bit
// scores), and comparing keys is the whole tie rule.
// A row is cut into tiles of 4096; a workgroup holds its tile's keys in registers, finds the tile's
// k-th largest key by a radix descent over LDS histograms and keeps the k keys at or above it.  The
// kept keys of all tiles are the next, k / 4096 times shorter, row; the last level sorts.
#include "alsmi_common.h"
#include "elem.h"

namespace alsmi {

constexpr int TR_THREADS = 256;
constexpr int TR_E = 16;                       // keys per thread
constexpr int TR_TILE = TR_THREADS * TR_E;     // 4096
constexpr int TR_MAX_K = 1024;

typedef unsigned __int128 u128;

template <typename T>
struct RowKey {  // 16- and 32-bit scores through their fp32 image
    typedef unsigned long long type;
    static constexpr int BITS = 64;
    static __device__ __forceinline__ type make(T s, unsigned index) {
        const unsigned b = __builtin_bit_cast(unsigned, (float)s);
        const unsigned image = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
        return ((type)image << 32) | (unsigned)~index;
    }
    static __device__ __forceinline__ T score(type k) {
        const unsigned i = (unsigned)(k >> 32);
        return (T)__builtin_bit_cast(float, (i & 0x80000000u) ? (i & 0x7fffffffu) : ~i);
    }
};
template <>
struct RowKey<double> {
    typedef u128 type;
    static constexpr int BITS = 96;
    static __device__ __forceinline__ type make(double s, unsigned index) {
        const unsigned long long b = __builtin_bit_cast(unsigned long long, s);
        const unsigned long long image = (b >> 63) ? ~b : (b | 0x8000000000000000ull);
        return ((type)image << 32) | (unsigned)~index;
    }
    static __device__ __forceinline__ double score(type k) {
        const unsigned long long i = (unsigned long long)(k >> 32);
        return __builtin_bit_cast(double, (i >> 63) ? (i & 0x7fffffffffffffffull) : ~i);
    }
};

// One tile: keys of `n` elements (scores, or keys left by the level before) starting at `first`.
// SORT: the only tile of its row; its k best are sorted and written out.
template <typename T, bool FROM_KEYS, bool SORT>
__global__ __launch_bounds__(TR_THREADS) void topk_rows_kernel(
    const T *__restrict__ scores, int64_t lds, const typename RowKey<T>::type *__restrict__ in,
    int64_t n, int k, unsigned tiles, typename RowKey<T>::type *__restrict__ kept,
    int32_t *__restrict__ items_out, T *__restrict__ scores_out) {
    typedef typename RowKey<T>::type key_t;
    __shared__ unsigned hist[256];
    __shared__ key_t sel[SORT ? TR_MAX_K : 1];
    __shared__ int bin_sh, above_sh, in_bin_sh, n_kept;
    const int tid = threadIdx.x;
    const unsigned r32 = blockIdx.x / tiles;
    const int64_t row = r32;
    const unsigned tile = blockIdx.x - r32 * tiles;
    const int64_t first = (int64_t)tile * TR_TILE;
    const int64_t left = n - first;
    const int count = left < TR_TILE ? (int)left : TR_TILE;
    key_t key[TR_E];
#pragma unroll
    for (int j = 0; j < TR_E; ++j) {
        const int i = j * TR_THREADS + tid;
        key[j] = 0;  // below every key: ~index is never 0
        if (i < count) {
            if constexpr (FROM_KEYS) key[j] = in[row * n + first + i];
            else key[j] = RowKey<T>::make(scores[row * lds + first + i], (unsigned)(first + i));
        }
    }
    // radix descent: `floor` = the smallest key kept
    key_t floor_key = 1;
    if (count > k) {
        key_t prefix = 0;
        int want = k;
        for (int shift = RowKey<T>::BITS - 8; shift >= 0; shift -= 8) {
            hist[tid] = 0;
            __syncthreads();
            const key_t high = shift + 8 >= RowKey<T>::BITS ? (key_t)0 : ~(key_t)0 << (shift + 8);
            int run_bin = -1;
            unsigned run = 0;
#pragma unroll
            for (int j = 0; j < TR_E; ++j) {
                if ((key[j] & high) != prefix) continue;
                const int b = (int)(key[j] >> shift) & 255;
                if (b != run_bin) {
                    if (run) atomicAdd(&hist[run_bin], run);
                    run_bin = b;
                    run = 0;
                }
                ++run;
            }
            if (run) atomicAdd(&hist[run_bin], run);
            __syncthreads();
            if (tid < 64) {
                // lane l holds bins 255 - 4l .. 252 - 4l; running count from the top
                unsigned h[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) sum += h[i] = hist[255 - 4 * tid - i];
                unsigned upto = sum;
#pragma unroll
                for (int off = 1; off < 64; off <<= 1) {
                    const unsigned o = __shfl_up(upto, off);
                    if (tid >= off) upto += o;
                }
                unsigned above = upto - sum;
                if (above < (unsigned)want && upto >= (unsigned)want) {
                    int i = 0;
                    while (above + h[i] < (unsigned)want) above += h[i++];
                    bin_sh = 255 - 4 * tid - i;
                    above_sh = (int)above;
                    in_bin_sh = (int)h[i];
                }
            }
            __syncthreads();
            prefix |= (key_t)bin_sh << shift;
            want -= above_sh;
            if (in_bin_sh == want) break;  // the whole bin is kept
        }
        floor_key = prefix;
    }
    if (tid == 0) n_kept = 0;
    __syncthreads();
    key_t *dst = SORT ? sel : kept + (row * tiles + tile) * k;
#pragma unroll
    for (int j = 0; j < TR_E; ++j)
        if (key[j] != 0 && key[j] >= floor_key) dst[atomicAdd(&n_kept, 1)] = key[j];
    __syncthreads();
    const int have = n_kept;
    if constexpr (!SORT) {
        for (int i = have + tid; i < k; i += TR_THREADS) dst[i] = 0;
    } else {
        int np2 = 1;
        while (np2 < k) np2 <<= 1;
        for (int i = have + tid; i < np2; i += TR_THREADS) sel[i] = 0;
        __syncthreads();
        for (int size = 2; size <= np2; size <<= 1)
            for (int stride = size >> 1; stride > 0; stride >>= 1) {
                for (int i = tid; i < np2 / 2; i += TR_THREADS) {
                    const int lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
                    const key_t a = sel[lo], b = sel[hi];
                    if ((a > b) != ((lo & size) == 0)) {
                        sel[lo] = b;
                        sel[hi] = a;
                    }
                }
                __syncthreads();
            }
        for (int i = tid; i < k; i += TR_THREADS) {
            items_out[row * k + i] = (int32_t)~(unsigned)sel[i];
            scores_out[row * k + i] = RowKey<T>::score(sel[i]);
        }
    }
}

static int64_t topk_tiles(int64_t n) { return (n + TR_TILE - 1) / TR_TILE; }

template <typename T>
static int run_topk_rows(int64_t n_rows, int64_t n_items, const void *scores, int64_t lds, int k,
                         int32_t *items_out, void *scores_out, void *workspace, hipStream_t st) {
    typedef typename RowKey<T>::type key_t;
    const T *s = static_cast<const T *>(scores);
    T *so = static_cast<T *>(scores_out);
    // keys of the first level, then levels alternate between the two halves of the workspace
    int64_t n = n_items, tiles = topk_tiles(n);
    key_t *a = static_cast<key_t *>(workspace), *b = a + n_rows * tiles * k;
    const dim3 block(TR_THREADS);
    auto grid = [&](int64_t t) { return dim3((unsigned)(t * n_rows)); };
    ALSMI_REQUIRE(tiles * n_rows <= INT32_MAX, "alsmi_topk_rows: too many rows x items");
    if (tiles == 1) {
        hipLaunchKernelGGL((topk_rows_kernel<T, false, true>), grid(1), block, 0, st, s, lds,
                           (const key_t *)nullptr, n, k, 1u, (key_t *)nullptr, items_out, so);
        ALSMI_HIP_CHECK(hipGetLastError());
        return ALSMI_OK;
    }
    hipLaunchKernelGGL((topk_rows_kernel<T, false, false>), grid(tiles), block, 0, st, s, lds,
                       (const key_t *)nullptr, n, k, (unsigned)tiles, a, (int32_t *)nullptr,
                       (T *)nullptr);
    ALSMI_HIP_CHECK(hipGetLastError());
    for (;;) {
        n = tiles * k;
        tiles = topk_tiles(n);
        if (tiles == 1) break;
        hipLaunchKernelGGL((topk_rows_kernel<T, true, false>), grid(tiles), block, 0, st, s, lds, a, n,
                           k, (unsigned)tiles, b, (int32_t *)nullptr, (T *)nullptr);
        ALSMI_HIP_CHECK(hipGetLastError());
        key_t *t = a;
        a = b;
        b = t;
    }
    hipLaunchKernelGGL((topk_rows_kernel<T, true, true>), grid(1), block, 0, st, s, lds, a, n, k, 1u,
                       (key_t *)nullptr, items_out, so);
    ALSMI_HIP_CHECK(hipGetLastError());
    return ALSMI_OK;
}

}  // namespace alsmi

extern "C" {

size_t alsmi_topk_rows_workspace_bytes(int dtype, int64_t n_rows, int64_t n_items, int k) {
    using namespace alsmi;
    if (dtype < ALSMI_F32 || dtype > ALSMI_BF16 || n_rows < 0 || n_items < 0 || k < 1 || k > TR_MAX_K)
        return 0;
    const int64_t t1 = topk_tiles(n_items);
    if (t1 <= 1) return 16;
    const int64_t t2 = topk_tiles(t1 * k);
    return (size_t)n_rows * (size_t)k * (size_t)(t1 + (t2 > 1 ? t2 : 0)) * (dtype == ALSMI_F64 ? 16 : 8) +
           16;
}

int alsmi_topk_rows(int dtype, int64_t n_rows, int64_t n_items, const void *scores, int64_t ld_scores,
                    int k, int32_t *items_out, void *scores_out, void *workspace, void *stream) {
    using namespace alsmi;
    ALSMI_REQUIRE(dtype >= ALSMI_F32 && dtype <= ALSMI_BF16, "alsmi_topk_rows: bad dtype %d", dtype);
    ALSMI_REQUIRE(n_rows >= 0 && n_rows <= INT32_MAX && n_items >= 0 && n_items <= INT32_MAX,
                  "alsmi_topk_rows: bad row or item count");
    ALSMI_REQUIRE(k >= 1 && k <= TR_MAX_K && k <= n_items,
                  "alsmi_topk_rows: need 1 <= k <= min(%d, n_items), got k=%d n_items=%lld", TR_MAX_K, k,
                  (long long)n_items);
    if (n_rows == 0) return ALSMI_OK;
    ALSMI_REQUIRE(ld_scores >= n_items || n_rows == 1, "alsmi_topk_rows: row stride below n_items");
    ALSMI_REQUIRE(scores && items_out && scores_out && workspace, "alsmi_topk_rows: null pointer");
    ALSMI_REQUIRE((uintptr_t)workspace % 16 == 0, "alsmi_topk_rows: workspace must be aligned to 16 bytes");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == ALSMI_F32)
        return run_topk_rows<float>(n_rows, n_items, scores, ld_scores, k, items_out, scores_out,
                                    workspace, st);
    if (dtype == ALSMI_F64)
        return run_topk_rows<double>(n_rows, n_items, scores, ld_scores, k, items_out, scores_out,
                                     workspace, st);
    if (dtype == ALSMI_F16)
        return run_topk_rows<_Float16>(n_rows, n_items, scores, ld_scores, k, items_out, scores_out,
                                       workspace, st);
    return run_topk_rows<__bf16>(n_rows, n_items, scores, ld_scores, k, items_out, scores_out, workspace,
                                 st);
}

}  // extern "C"
