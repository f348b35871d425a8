// The k largest scores of every row of a score block, best first, ties to the lowest index.
//
// Scores are ranked through the order-preserving integer image of their bits joined with the
// complement of their index, up to 96 bits.  These keys are all different, so "the k-th
// largest" is one element however many scores are equal (rows that a mask left mostly at -inf, 16-bit
// scores), comparing keys is the whole tie rule, and any set of candidates can be merged in any
// order.  0 is below every key.
//
// Small k: a wave keeps its k best, sorted, one per lane, and streams over its part of the row: a key at
//   or below the k-th best is dropped by one comparison, the few others wait in LDS until 64 of them
//   are sorted and merged into the list at once.  Four waves per workgroup, as many workgroups per row
//   as fill the chip; a second launch merges their lists.  Many rows take the time of their reads and
//   some more for sorting and merging hits (1024 x 26744 fp32, k = 10: 23.4 us, 4.7 TB/s; 18.8
//   without hits, 14.7 for the reads alone), one row that of two launches (1 x 1000000: 14 us).
// Larger k: a workgroup of 512 threads keeps the k best of its part of the row: of the first 8192 keys,
//   held in registers, it finds the k-th largest by a radix descent over LDS histograms (2048 bins
//   a digit), from then on only keys above it are looked at again.  Parts as many as run at once;
//   the kept keys of a row's parts are the next, much shorter, row.  The last level sorts.  Bound by
//   the latencies of the descent and the sort (1024 x 26744 fp32, k = 100: 44 us, 1000: 70; 37 x
//   100003 bf16, k = 1000: 30).
#include "alsmi_common.h"
#include "elem.h"

#include <algorithm>
#include <type_traits>
#include <utility>

namespace alsmi {

constexpr int TR_MAX_K = 1024;
constexpr int TR_LIST = 64;         // the longest list one wave keeps,
constexpr int TR_FEW = 24;          // and the longest kept whatever the rows
constexpr int TR_CHUNK = 1024;      // keys a wave looks at per turn, 16 per lane
constexpr int TR_PART = 4 * TR_CHUNK;
constexpr int TR_THREADS = 512;     // larger k: threads of a workgroup, keys they look at per turn,
constexpr int TR_TILE = 8192;
constexpr int TR_LAST = 16384;      // keys of a last turn by 1024 threads,
constexpr int TR_GROUPS = 1024;     // and workgroups that a launch of few rows is cut into

typedef unsigned __int128 u128;

template <typename T>
struct RowKey {  // fp32: 32 bits of image, 32 of index
    typedef unsigned long long type;
    typedef unsigned image_t;
    static constexpr int BITS = 64;
    static __device__ __forceinline__ image_t image(T s) {
        const unsigned b = __builtin_bit_cast(unsigned, s);
        return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
    }
    static __device__ __forceinline__ T score(image_t i) {
        return __builtin_bit_cast(T, (i & 0x80000000u) ? (i & 0x7fffffffu) : ~i);
    }
};
struct RowKey16 {  // fp16, bf16: 16 bits of image
    typedef unsigned long long type;
    typedef unsigned image_t;
    static constexpr int BITS = 48;
    static __device__ __forceinline__ image_t image(unsigned short b) {
        return (b ^ ((unsigned)((int)(short)b >> 31) | 0x8000u)) & 0xffffu;
    }
    static __device__ __forceinline__ unsigned short bits(image_t i) {
        return (unsigned short)((i & 0x8000u) ? (i & 0x7fffu) : ~i);
    }
};
template <>
struct RowKey<_Float16> : RowKey16 {
    static __device__ __forceinline__ image_t image(_Float16 s) {
        return RowKey16::image(__builtin_bit_cast(unsigned short, s));
    }
    static __device__ __forceinline__ _Float16 score(image_t i) {
        return __builtin_bit_cast(_Float16, bits(i));
    }
};
template <>
struct RowKey<__bf16> : RowKey16 {
    static __device__ __forceinline__ image_t image(__bf16 s) {
        return RowKey16::image(__builtin_bit_cast(unsigned short, s));
    }
    static __device__ __forceinline__ __bf16 score(image_t i) { return __builtin_bit_cast(__bf16, bits(i)); }
};
template <>
struct RowKey<double> {
    typedef u128 type;
    typedef unsigned long long image_t;
    static constexpr int BITS = 96;
    static __device__ __forceinline__ image_t image(double s) {
        const unsigned long long b = __builtin_bit_cast(unsigned long long, s);
        return b ^ ((unsigned long long)((long long)b >> 63) | 0x8000000000000000ull);
    }
    static __device__ __forceinline__ double score(image_t i) {
        return __builtin_bit_cast(double, (i >> 63) ? (i & 0x7fffffffffffffffull) : ~i);
    }
};

// Where a launch reads: a row of scores, or the keys that the level before kept of it.
template <typename T, bool FROM_KEYS>
struct KeySource {
    typedef typename RowKey<T>::type key_t;
    typedef typename std::conditional<FROM_KEYS, key_t, T>::type raw_t;
    const raw_t *data;
    int64_t ld;  // row stride
    int64_t n;
    // N elements of a row from `at` on; those at and behind `end` are not read
    template <int N>
    static __device__ __forceinline__ void load(raw_t (&v)[N], const raw_t *row, int64_t at, int64_t end) {
        if constexpr (sizeof(raw_t) == 16) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = at + i < end ? row[at + i] : (raw_t)0;
        } else {
            typedef raw_t vec_t __attribute__((ext_vector_type(N), aligned(sizeof(raw_t))));
            if (at + N <= end) {
                const vec_t w = *reinterpret_cast<const vec_t *>(row + at);
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = w[i];
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = at + i < end ? row[at + i] : (raw_t)0;
            }
        }
    }
    typedef typename RowKey<T>::image_t image_t;
    static __device__ __forceinline__ image_t image(raw_t v) {
        if constexpr (FROM_KEYS) return (image_t)(v >> 32);
        else return RowKey<T>::image(v);
    }
    // the key of element `at`; 0 at and behind `end`
    static __device__ __forceinline__ key_t key(raw_t v, int64_t at, int64_t end) {
        if constexpr (FROM_KEYS) return v;
        else return at < end ? ((key_t)RowKey<T>::image(v) << 32) | (unsigned)~(unsigned)at : (key_t)0;
    }
};

// The value of lane (lane ^ MASK).  All masks the sorts use are vector instructions (a shuffle through
// LDS takes some ten times as long): permutations of 4 lanes, mirrors of 8 and 16, a rotation of 16
// by 8, and the swaps of rows of 16 and halves of 32.
template <int MASK>
__device__ __forceinline__ unsigned lane_xor(unsigned x, int lane) {
    auto dpp = [](unsigned v, auto ctrl) {
        return (unsigned)__builtin_amdgcn_mov_dpp((int)v, decltype(ctrl)::value, 0xf, 0xf, true);
    };
    if constexpr (MASK == 1) return dpp(x, std::integral_constant<int, 0xb1>{});
    else if constexpr (MASK == 2) return dpp(x, std::integral_constant<int, 0x4e>{});
    else if constexpr (MASK == 3) return dpp(x, std::integral_constant<int, 0x1b>{});
    else if constexpr (MASK == 7) return dpp(x, std::integral_constant<int, 0x141>{});
    else if constexpr (MASK == 15) return dpp(x, std::integral_constant<int, 0x140>{});
    else if constexpr (MASK == 8) return dpp(x, std::integral_constant<int, 0x128>{});
    else if constexpr (MASK == 4) return lane_xor<3>(lane_xor<7>(x, lane), lane);
    else if constexpr (MASK == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        return (lane & 16) ? r[0] : r[1];
    } else if constexpr (MASK == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        return (lane & 32) ? r[0] : r[1];
    } else {
        static_assert(MASK == 31 || MASK == 63, "mask of no sort");
        return lane_xor<MASK == 63 ? 31 : 15>(lane_xor<MASK == 63 ? 32 : 16>(x, lane), lane);
    }
}
template <int MASK>
__device__ __forceinline__ unsigned long long key_xor(unsigned long long k, int lane) {
    return ((unsigned long long)lane_xor<MASK>((unsigned)(k >> 32), lane) << 32) |
           lane_xor<MASK>((unsigned)k, lane);
}
template <int MASK>
__device__ __forceinline__ u128 key_xor(u128 k, int lane) {  // (96 bits)
    return ((u128)lane_xor<MASK>((unsigned)(k >> 64), lane) << 64) |
           key_xor<MASK>((unsigned long long)k, lane);
}
__device__ __forceinline__ unsigned long long lane_key(unsigned long long k, int lane) {
    return ((unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(k >> 32), lane) << 32) |
           (unsigned)__builtin_amdgcn_readlane((int)k, lane);
}
__device__ __forceinline__ u128 lane_key(u128 k, int lane) {
    return ((u128)lane_key((unsigned long long)(k >> 64), lane) << 64) |
           lane_key((unsigned long long)k, lane);
}

// One step of a sort, largest first: of lanes l and l ^ MASK the one without MASK's top bit keeps the
// larger key.
template <int MASK, typename K>
__device__ __forceinline__ K sort_step(K k, int lane) {
    constexpr int TOP = MASK >= 32 ? 32 : MASK >= 16 ? 16 : MASK >= 8 ? 8 : MASK >= 4 ? 4 : MASK >= 2 ? 2 : 1;
    const K o = key_xor<MASK>(k, lane);
    return (o > k) != ((lane & TOP) != 0) ? o : k;
}
// A bitonic sequence of the 64 lanes put in order; all of them sorted.  (A sorted run meets the mirror
// image of the next one, so every run is sorted the same way.)
template <typename K>
__device__ __forceinline__ K wave_merge(K k, int lane) {
    k = sort_step<32>(k, lane);
    k = sort_step<16>(k, lane);
    k = sort_step<8>(k, lane);
    k = sort_step<4>(k, lane);
    k = sort_step<2>(k, lane);
    return sort_step<1>(k, lane);
}
template <typename K>
__device__ __forceinline__ K wave_sort(K k, int lane) {
    k = sort_step<1>(k, lane);
    k = sort_step<3>(k, lane);
    k = sort_step<1>(k, lane);
    k = sort_step<7>(k, lane);
    k = sort_step<2>(k, lane);
    k = sort_step<1>(k, lane);
    k = sort_step<15>(k, lane);
    k = sort_step<4>(k, lane);
    k = sort_step<2>(k, lane);
    k = sort_step<1>(k, lane);
    k = sort_step<31>(k, lane);
    k = sort_step<8>(k, lane);
    k = sort_step<4>(k, lane);
    k = sort_step<2>(k, lane);
    k = sort_step<1>(k, lane);
    k = sort_step<63>(k, lane);
    k = sort_step<16>(k, lane);
    k = sort_step<8>(k, lane);
    k = sort_step<4>(k, lane);
    k = sort_step<2>(k, lane);
    return sort_step<1>(k, lane);
}
// the best 64 of two sorted lists, sorted
template <typename K>
__device__ __forceinline__ K wave_join(K list, K other, int lane) {
    const K back = key_xor<63>(other, lane);
    return wave_merge(back > list ? back : list, lane);
}

// SHORT: rows of at most one chunk, a wave each, four to a workgroup (262144 x 100 fp32, k = 10: 0.29 ms
// instead of 1.48).
template <typename T, bool FROM_KEYS, bool SHORT>
__global__ __launch_bounds__(256) void topk_list_kernel(KeySource<T, FROM_KEYS> src, int64_t n_rows, int k,
                                                        unsigned parts, int64_t part_len,
                                                        typename RowKey<T>::type *__restrict__ kept,
                                                        int32_t *__restrict__ items_out,
                                                        T *__restrict__ scores_out) {
    typedef typename RowKey<T>::type key_t;
    // elements per load (16 bytes), loads per chunk
    constexpr int VEC = FROM_KEYS ? 16 / (int)sizeof(key_t) : 16 / (int)sizeof(T);
    constexpr int LOADS = 16 / VEC;
    __shared__ key_t waiting_sh[4][TR_LIST + TR_CHUNK];
    __shared__ key_t bounds[4][TR_LIST], lists[4][TR_LIST];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned r32 = SHORT ? blockIdx.x * 4 + wave : blockIdx.x / parts;
    const int64_t row = r32;
    if (SHORT && row >= n_rows) return;
    const unsigned part = SHORT ? 0 : blockIdx.x - r32 * parts;
    const int64_t first = (int64_t)part * part_len;
    const int64_t end = first + part_len < src.n ? first + part_len : src.n;
    volatile key_t *waiting = waiting_sh[wave];  // (one wave's reads and writes of LDS keep their order)
    key_t list = 0;      // the wave's best so far, best in lane 0
    key_t floor_key = 0; // keys at or below it are out
    int n_waiting = 0;
    auto flush = [&]() {
        const int m = n_waiting < TR_LIST ? n_waiting : TR_LIST;
        n_waiting -= m;
        key_t v = 0;
        if (lane < m) v = waiting[n_waiting + lane];
        list = wave_join(list, wave_sort(v, lane), lane);
        const key_t kth = lane_key(list, k - 1);
        floor_key = kth > floor_key ? kth : floor_key;
    };
    typedef KeySource<T, FROM_KEYS> source;
    const typename source::raw_t *data = src.data + row * src.ld;
    typename source::raw_t raw[LOADS][VEC];
    auto fetch = [&](int64_t at) {
        if (at + TR_CHUNK <= end) {  // (the whole wave alike: plain loads, all in flight together)
#pragma unroll
            for (int j = 0; j < LOADS; ++j)
                source::load(raw[j], data + at + (j * 64 + lane) * VEC, 0, VEC);
        } else {
#pragma unroll
            for (int j = 0; j < LOADS; ++j) source::load(raw[j], data, at + (j * 64 + lane) * VEC, end);
        }
    };
    const int64_t start = SHORT ? 0 : first + wave * TR_CHUNK;
    fetch(start);
    {
        // a first bound: the k-th largest of the lanes' largest of the waves' first chunks
        key_t top = 0;
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const key_t x = source::key(raw[j][i], start + (j * 64 + lane) * VEC + i, end);
                top = x > top ? x : top;
            }
        top = wave_sort(top, lane);
        if constexpr (!SHORT) {
            bounds[wave][lane] = top;
            __syncthreads();
#pragma unroll 1
            for (int w = 1; w < 4; ++w) top = wave_join(top, (key_t)bounds[(wave + w) & 3][lane], lane);
        }
        const key_t kth = lane_key(top, k - 1);
        floor_key = kth ? kth - 1 : 0;
    }
    for (int64_t at = start; at < end; at += 4 * TR_CHUNK) {
        typename source::raw_t now[LOADS][VEC];
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) now[j][i] = raw[j][i];
        // (the next chunk is on its way while this one is looked at)
        if (!SHORT && at + 4 * TR_CHUNK < end) fetch(at + 4 * TR_CHUNK);
        auto key_at = [&](int j, int i) {
            return source::key(now[j][i], at + (j * 64 + lane) * VEC + i, end);
        };
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            // most loads hold nothing: one look at the largest score of a lane, whole keys only then
            // (elements behind the end count as whatever they are read as, and are no hits)
            typename source::image_t top = source::image(now[j][0]);
#pragma unroll
            for (int i = 1; i < VEC; ++i) {
                const typename source::image_t x = source::image(now[j][i]);
                top = x > top ? x : top;
            }
            if (__ballot(top >= (typename source::image_t)(floor_key >> 32)) == 0) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const key_t x = key_at(j, i);
                const bool hit = x > floor_key;
                const unsigned long long m = __ballot(hit);
                if (m == 0) continue;
                if (hit) waiting[n_waiting + __popcll(m & ((1ull << lane) - 1ull))] = x;
                n_waiting += __popcll(m);
            }
        }
        // (in one place: unrolled into every load this was 60 KB of code, and fetching it the
        // largest part of a small launch)
        const bool last = at + 4 * TR_CHUNK >= end;
        while (n_waiting >= TR_LIST || (last && n_waiting > 0)) flush();
    }
    if constexpr (!SHORT) {
        lists[wave][lane] = list;
        __syncthreads();
        if (wave > 0) return;
#pragma unroll 1
        for (int w = 1; w < 4; ++w) list = wave_join(list, (key_t)lists[w][lane], lane);
    }
    if (lane >= k) return;
    if (parts > 1) {
        kept[(row * parts + part) * k + lane] = list;
    } else {
        items_out[row * k + lane] = (int32_t)~(unsigned)list;
        scores_out[row * k + lane] = RowKey<T>::score((typename RowKey<T>::image_t)(list >> 32));
    }
}

// ---- larger k ------------------------------------------------------------------------------------
// Sum over lanes 0 .. lane.
__device__ __forceinline__ unsigned wave_prefix(unsigned x) {
    auto add = [&](auto ctrl, auto rows) {
        x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, decltype(rows)::value,
                                                   0xf, false);
    };
    add(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});  // from 1 lane below,
    add(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});  // 2, 4, 8 inside a row
    add(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
    add(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
    add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // row ends to rows 1, 3
    add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // the lower half's end
    return x;
}

// The smallest of the k largest keys of a workgroup (THREADS x E keys of at most `bits` bits in
// registers, all different but for zeros, which stand for none), by digits of 11 bits from the top; 0
// if there are fewer than k.  A pass costs its atomics and two barriers: every wave reads the whole histogram
// and finds the digit by itself (one wave, or sums by thread and prefix sums over the workgroup,
// with more barriers, took longer), and the other of two histograms is cleared meanwhile.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
constexpr int TR_DIGIT = 11, TR_BINS = 1 << TR_DIGIT;
template <typename K, int THREADS, int E, int HELD>
__device__ __forceinline__ K kth_key(const K (&key)[HELD], int k, int bits, u32x4 (&hist4)[2][TR_BINS / 4]) {
    constexpr int DIGIT = TR_DIGIT, BINS = TR_BINS, LANE_BINS = BINS / 64;
    const int tid = threadIdx.x, lane = tid & 63;
    K prefix = 0;
    unsigned want = k;
    for (int i = tid; i < BINS / 4; i += THREADS) hist4[0][i] = u32x4{0, 0, 0, 0};
    __syncthreads();
    int turn = 0;
    for (int high = bits; high > 0; high -= DIGIT, turn ^= 1) {  // bits [low, high) of the keys
        unsigned *hist = reinterpret_cast<unsigned *>(hist4[turn]);
        const int low = high > DIGIT ? high - DIGIT : 0;
        const unsigned mask = (1u << (high - low)) - 1u;
        const K upper = ~(K)0 << high;
        // scores share their leading bits: a thread adds up a run of equal digits first
        int run_bin = -1;
        unsigned run = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            if ((key[j] & upper) != prefix || key[j] == 0) continue;
            const int b = (int)((unsigned)(key[j] >> low) & mask);
            if (b != run_bin) {
                if (run) atomicAdd(&hist[run_bin], run);
                run_bin = b;
                run = 0;
            }
            ++run;
        }
        if (run) atomicAdd(&hist[run_bin], run);
        for (int i = tid; i < BINS / 4; i += THREADS) hist4[turn ^ 1][i] = u32x4{0, 0, 0, 0};
        __syncthreads();
        // lane l: the 32 bins below BINS - 32 l (its reads start at another place than its neighbours',
        // or all lanes would meet in the same banks)
        unsigned sum = 0;
#pragma unroll
        for (int i = 0; i < LANE_BINS / 4; ++i) {
            const u32x4 h = hist4[turn][(63 - lane) * (LANE_BINS / 4) + ((i + lane) & (LANE_BINS / 4 - 1))];
            sum += h[0] + h[1] + h[2] + h[3];
        }
        unsigned upto = wave_prefix(sum);
        unsigned long long found = __ballot(upto >= want);
        if (found == 0) return 0;
        const int owner = __builtin_ctzll(found);
        unsigned above = (unsigned)__builtin_amdgcn_readlane((int)(upto - sum), owner);
        // and the bin among the owner's
        const int top = BINS - LANE_BINS * owner - 1;
        const unsigned h = lane < LANE_BINS ? hist[top - lane] : 0u;
        upto = above + wave_prefix(h);
        found = __ballot(upto >= want);
        const int at = __builtin_ctzll(found);
        above = (unsigned)__builtin_amdgcn_readlane((int)(upto - h), at);
        const unsigned in_bin = (unsigned)__builtin_amdgcn_readlane((int)h, at);
        prefix |= (K)(unsigned)(top - at) << low;
        want -= above;
        if (in_bin == want) break;  // the whole bin is in
        __syncthreads();            // (the other histogram is clear, this one read)
    }
    return prefix;
}

// Workgroup (row, part) keeps the k best of its part of the row and writes them to `kept`, or, SORT, the
// whole row's sorted.  It walks the part in tiles of TILE keys: those above the k-th best so far
// are appended to the kept ones in LDS (one barrier a tile), and where these would be more than
// 2 TR_MAX_K, as for the first tile, kept ones and tile are cut down to the best k together.
// Keys here are image << index_bits | n_items - index, never 0.
template <typename T, bool FROM_KEYS, bool SORT, int THREADS, int TILE>
__global__ __launch_bounds__(THREADS) void topk_tile_kernel(KeySource<T, FROM_KEYS> src, int k,
                                                               unsigned n_items, int index_bits,
                                                               unsigned parts, int64_t part_len,
                                                               typename RowKey<T>::type *__restrict__ kept,
                                                               int32_t *__restrict__ items_out,
                                                               T *__restrict__ scores_out) {
    typedef typename RowKey<T>::type key_t;
    typedef KeySource<T, FROM_KEYS> source;
    constexpr int E = TILE / THREADS;
    constexpr int VEC = 16 / (int)sizeof(typename source::raw_t);
    constexpr int ROOM = 2 * TR_MAX_K;
    constexpr int KEEP = ROOM / THREADS, SORTED = TR_MAX_K / THREADS;  // keys of a thread of these
    __shared__ key_t sel[ROOM];
    __shared__ u32x4 hist[2][TR_BINS / 4];
    __shared__ int added[3];  // keys added by a step; the one after the next step's is cleared meanwhile
    const int tid = threadIdx.x, lane = tid & 63;
    const unsigned r32 = blockIdx.x / parts;
    const int64_t row = r32;
    const unsigned part = blockIdx.x - r32 * parts;
    const int64_t first = (int64_t)part * part_len;
    const int64_t end = first + part_len < src.n ? first + part_len : src.n;
    const typename source::raw_t *data = src.data + row * src.ld;
    key_t floor_key = 0;  // keys at or below it are out
    int have = 0, step = 0;
    key_t key[E + KEEP];  // a tile's, and of the kept ones when these are cut down
    // the first N keys that are above floor_key go behind the `have` kept ones; how many there are
    auto append = [&](auto n, auto put) __attribute__((always_inline)) {
        constexpr int N = decltype(n)::value;
        unsigned mine = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) mine += key[j] > floor_key;
        int *count = &added[step];
        if (__any(mine)) {
            const unsigned upto = wave_prefix(mine);
            int place = 0;
            if (lane == 63) place = atomicAdd(count, (int)upto);
            place = have + __builtin_amdgcn_readlane(place, 63) + (int)(upto - mine);
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (key[j] > floor_key) put(place++, key[j]);
        }
        __syncthreads();
        const int got = *count;
        step = step == 2 ? 0 : step + 1;
        if (tid == 0) added[step == 2 ? 0 : step + 1] = 0;
        return got;
    };
    auto to_sel = [&](int place, key_t x) {
        if (place < ROOM) sel[place] = x;
    };
    const int bits = RowKey<T>::BITS - 32 + index_bits;
    // kept ones and key[0 .. E) cut down to the k best
    auto cut = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < KEEP; ++i)
            key[E + i] = i * THREADS + tid < have ? sel[i * THREADS + tid] : (key_t)0;
        const key_t kth = kth_key<key_t, THREADS, E + KEEP>(key, k, bits, hist);
        floor_key = kth ? kth - 1 : 0;
        have = 0;
        __syncthreads();
        have = append(std::integral_constant<int, E + KEEP>{}, to_sel);
        floor_key = kth;
    };
    typename source::raw_t raw[E / VEC][VEC];
    auto fetch = [&](int64_t at0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < E / VEC; ++j) source::load(raw[j], data, at0 + (j * THREADS + tid) * VEC, end);
    };
    fetch(first);
    if (tid < 3) added[tid] = 0;
    __syncthreads();
    for (int64_t at0 = first; at0 < end; at0 += TILE) {
#pragma unroll
        for (int j = 0; j < E / VEC; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int64_t at = at0 + (j * THREADS + tid) * VEC + i;
                if constexpr (FROM_KEYS) key[j * VEC + i] = raw[j][i];
                else
                    key[j * VEC + i] = at < end ? (key_t)RowKey<T>::image(raw[j][i]) << index_bits |
                                                      (n_items - (unsigned)at)
                                                : (key_t)0;
            }
        if (at0 + TILE < end) fetch(at0 + TILE);  // (on its way while this one is looked at)
        if constexpr (!SORT) {
            if (first + TILE >= end) {  // the only tile: straight from the registers
                key_t *dst = kept + (row * parts + part) * k;
                const key_t kth = kth_key<key_t, THREADS, E>(key, k, bits, hist);
                floor_key = kth ? kth - 1 : 0;
                have = append(std::integral_constant<int, E>{}, [&](int place, key_t x) { dst[place] = x; });
                for (int i = have + tid; i < k; i += THREADS) dst[i] = 0;
                return;
            }
        }
        // (before there is a bound every key of a tile would be added)
        if (floor_key != 0 || have + (end - at0) <= ROOM) {
            const int got = append(std::integral_constant<int, E>{}, to_sel);
            if (have + got <= ROOM) {
                have += got;
                continue;
            }
        }
        cut();
    }
    if (have > k) {
#pragma unroll
        for (int j = 0; j < E; ++j) key[j] = 0;
        cut();
    }
    if constexpr (!SORT) {
        key_t *dst = kept + (row * parts + part) * k;
        for (int i = tid; i < k; i += THREADS) dst[i] = i < have ? sel[i] : (key_t)0;
    } else {
        // sorted by wave, then runs of 64, 128, ... meet the mirror image of the next run; steps within a
        // wave go through the lanes, the others through LDS
        key_t mine[SORTED];
#pragma unroll
        for (int r = 0; r < SORTED; ++r) {
            const int i = r * THREADS + tid;
            mine[r] = wave_sort(i < have ? sel[i] : (key_t)0, lane);
        }
        for (int size = 128; size < 2 * k; size <<= 1) {  // (runs behind the k-th key hold zeros)
            int mask = size - 1;
            for (int top = size >> 1; top >= 64; top >>= 1) {
                __syncthreads();
#pragma unroll
                for (int r = 0; r < SORTED; ++r) sel[r * THREADS + tid] = mine[r];
                __syncthreads();
#pragma unroll
                for (int r = 0; r < SORTED; ++r) {
                    const int i = r * THREADS + tid;
                    const key_t o = sel[i ^ mask];
                    mine[r] = (o > mine[r]) != ((i & top) != 0) ? o : mine[r];
                }
                mask = top >> 1;
            }
#pragma unroll
            for (int r = 0; r < SORTED; ++r) mine[r] = wave_merge(mine[r], lane);
        }
#pragma unroll
        for (int r = 0; r < SORTED; ++r) {
            const int i = r * THREADS + tid;
            if (i >= k) continue;
            items_out[row * k + i] =
                (int32_t)(n_items - ((unsigned)mine[r] & (0xffffffffu >> (32 - index_bits))));
            scores_out[row * k + i] =
                RowKey<T>::score((typename RowKey<T>::image_t)(mine[r] >> index_bits));
        }
    }
}

// ---- launches ------------------------------------------------------------------------------------
// Lists: workgroups per row, so that a launch has about TR_GROUPS, at least 4096 keys each.
static int64_t list_parts(int64_t n_rows, int64_t n_items, int64_t &part_len) {
    const int64_t most = (n_items + TR_PART - 1) / TR_PART;
    int64_t parts = most <= 4 ? 1 : TR_GROUPS / n_rows;  // (a second launch costs more than four turns)
    parts = parts < 1 ? 1 : (parts > most ? most : parts);
    part_len = ((n_items + parts - 1) / parts + TR_PART - 1) / TR_PART * TR_PART;
    return (n_items + part_len - 1) / part_len;
}
// Tiles: workgroups per row, so that a launch has about TR_GROUPS, of whole tiles.
static int64_t tile_parts(int64_t n_rows, int64_t n, int64_t &part_len) {
    const int64_t most = (n + TR_TILE - 1) / TR_TILE;
    int64_t parts = most <= 2 ? 1 : TR_GROUPS / n_rows;  // (a second launch costs more than a second tile)
    parts = parts < 1 ? 1 : (parts > most ? most : parts);
    part_len = (most + parts - 1) / parts * TR_TILE;
    return (n + part_len - 1) / part_len;
}
// Which of the two forms: sorted lists take 29 us against 42 for 1024 x 26744 fp32 and k = 64, 13.4
// against 21 for 512 x 16384 and k = 32, but 28 against 18 for 1 x 1000000 and k = 64, 17.5 against 14 for
// 1 x 100000 and k = 32 (14.4 either way for k = 10): a row of many parts has many lists to merge.
static bool by_lists(int64_t n_rows, int64_t n_items, int k) {
    return k <= TR_FEW || (k <= TR_LIST && (n_rows > 128 || n_items <= 4 * TR_PART));
}
// Rows that are worked on at once: a launch has fewer than 2^32 threads.  Their number decides over the
// parts of a row for a smaller rest as well, so that the workspace does.
static int64_t batch_rows(int64_t n_rows) { return std::min(n_rows, (int64_t)1 << 21); }

template <typename T>
static int run_lists(int64_t n_rows, int64_t batch, const KeySource<T, false> &src, int k, int32_t *items_out,
                     T *scores_out, typename RowKey<T>::type *kept, hipStream_t st) {
    typedef typename RowKey<T>::type key_t;
    if (src.n <= TR_CHUNK) {
        hipLaunchKernelGGL((topk_list_kernel<T, false, true>), dim3((unsigned)((n_rows + 3) / 4)), dim3(256),
                           0, st, src, n_rows, k, 1u, src.n, (key_t *)nullptr, items_out, scores_out);
        ALSMI_HIP_CHECK(hipGetLastError());
        return ALSMI_OK;
    }
    int64_t part_len = 0;
    const int64_t parts = list_parts(batch, src.n, part_len);
    hipLaunchKernelGGL((topk_list_kernel<T, false, false>), dim3((unsigned)(parts * n_rows)), dim3(256), 0,
                       st, src, n_rows, k, (unsigned)parts, part_len, kept, items_out, scores_out);
    ALSMI_HIP_CHECK(hipGetLastError());
    if (parts == 1) return ALSMI_OK;
    const int64_t n = parts * k;
    const KeySource<T, true> left = {kept, n, n};
    hipLaunchKernelGGL((topk_list_kernel<T, true, false>), dim3((unsigned)n_rows), dim3(256), 0, st, left,
                       n_rows, k, 1u, (n + TR_PART - 1) / TR_PART * TR_PART, (key_t *)nullptr, items_out,
                       scores_out);
    ALSMI_HIP_CHECK(hipGetLastError());
    return ALSMI_OK;
}

// The level that sorts: a workgroup per row.  Rows of one to two tiles go as one larger one while
// there are not enough of them to fill the chip (200 x 16384 fp32, k = 100: 13.1 us instead of 15.6;
// 1024 x 16384: 44 instead of 36).
template <typename T, bool FROM_KEYS>
static int run_last(int64_t n_rows, const KeySource<T, FROM_KEYS> &src, int k, unsigned n_items, int index_bits,
                    int64_t part_len, int32_t *items_out, T *scores_out, hipStream_t st) {
    typedef typename RowKey<T>::type key_t;
    auto kernel = topk_tile_kernel<T, FROM_KEYS, true, TR_THREADS, TR_TILE>;
    int threads = TR_THREADS;
    if constexpr (sizeof(key_t) == 8) {  // (16 keys of 96 bits are too many registers for 1024 threads)
        if (src.n > TR_TILE && src.n <= TR_LAST && n_rows <= 512) {
            kernel = topk_tile_kernel<T, FROM_KEYS, true, TR_MAX_K, TR_LAST>;
            threads = TR_MAX_K;
        }
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)n_rows), dim3(threads), 0, st, src, k, n_items, index_bits, 1u,
                       part_len, (key_t *)nullptr, items_out, scores_out);
    ALSMI_HIP_CHECK(hipGetLastError());
    return ALSMI_OK;
}

template <typename T>
static int run_tiles(int64_t n_rows, int64_t batch, const KeySource<T, false> &src, int k, int32_t *items_out,
                     T *scores_out, typename RowKey<T>::type *kept, hipStream_t st) {
    typedef typename RowKey<T>::type key_t;
    int index_bits = 1;
    while (src.n >> index_bits) ++index_bits;
    int64_t part_len = 0, parts = tile_parts(batch, src.n, part_len);
    const dim3 block(TR_THREADS);
    if (parts == 1) {
        return run_last<T, false>(n_rows, src, k, (unsigned)src.n, index_bits, part_len, items_out, scores_out,
                                  st);
    }
    hipLaunchKernelGGL((topk_tile_kernel<T, false, false, TR_THREADS, TR_TILE>),
                       dim3((unsigned)(parts * n_rows)), block, 0, st, src, k, (unsigned)src.n, index_bits,
                       (unsigned)parts, part_len, kept, (int32_t *)nullptr, (T *)nullptr);
    ALSMI_HIP_CHECK(hipGetLastError());
    // the levels alternate between the two parts of the workspace
    key_t *from = kept, *to = kept + n_rows * parts * k;
    for (;;) {
        const int64_t n = parts * k;
        const KeySource<T, true> left = {from, n, n};
        parts = tile_parts(batch, n, part_len);
        if (parts == 1) {
            return run_last<T, true>(n_rows, left, k, (unsigned)src.n, index_bits, part_len, items_out,
                                     scores_out, st);
        }
        hipLaunchKernelGGL((topk_tile_kernel<T, true, false, TR_THREADS, TR_TILE>),
                           dim3((unsigned)(parts * n_rows)), block, 0, st, left, k, (unsigned)src.n,
                           index_bits, (unsigned)parts, part_len, to, (int32_t *)nullptr, (T *)nullptr);
        ALSMI_HIP_CHECK(hipGetLastError());
        std::swap(from, to);
    }
}

template <typename T>
static int run_topk_rows(int64_t n_rows, int64_t n_items, const void *scores, int64_t ld, int k,
                         int32_t *items_out, void *scores_out, void *workspace, hipStream_t st) {
    typedef typename RowKey<T>::type key_t;
    T *so = static_cast<T *>(scores_out);
    key_t *kept = static_cast<key_t *>(workspace);
    const int64_t batch = batch_rows(n_rows);  // (the workspace serves one batch after the other)
    const bool lists = by_lists(n_rows, n_items, k);
    for (int64_t lo = 0; lo < n_rows; lo += batch) {
        const int64_t rows = std::min(n_rows - lo, batch);
        const KeySource<T, false> src = {static_cast<const T *>(scores) + lo * ld, ld, n_items};
        const int status = lists ? run_lists<T>(rows, batch, src, k, items_out + lo * k, so + lo * k, kept, st)
                                 : run_tiles<T>(rows, batch, src, k, items_out + lo * k, so + lo * k, kept, st);
        if (status != ALSMI_OK) return status;
    }
    return ALSMI_OK;
}

}  // namespace alsmi

extern "C" {

size_t alsmi_topk_rows_workspace_bytes(int dtype, int64_t n_rows, int64_t n_items, int k) {
    using namespace alsmi;
    if (dtype < ALSMI_F32 || dtype > ALSMI_BF16 || n_rows < 0 || n_items < 0 || k < 1 || k > TR_MAX_K)
        return 0;
    if (n_rows == 0 || n_items == 0) return 16;
    // enough for any number of rows up to n_rows, of items up to n_items and for any smaller k: rows of up
    // to 16384 items are not cut, the parts of others at most TR_GROUPS (once more for the next level)
    if (n_items <= 4 * TR_PART) return 16;
    const int64_t parts = std::min<int64_t>(TR_GROUPS, n_rows * ((n_items + TR_PART - 1) / TR_PART));
    return (size_t)parts * (size_t)k * (k > TR_FEW ? 2 : 1) * (dtype == ALSMI_F64 ? 16 : 8) + 16;
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
