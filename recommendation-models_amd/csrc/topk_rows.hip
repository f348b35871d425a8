// The k largest scores of every row of a score block, best first, ties to the lowest index.
//
// Scores are ranked through the order-preserving integer image of their bits joined with the
// complement of their index: (image << 32) | ~index, 48, 64 or 96 bits.  These keys are all different, so "the k-th
// largest" is one element however many scores are equal (rows that a mask left mostly at -inf, 16-bit
// scores), comparing keys is the whole tie rule, and any set of candidates can be merged in any
// order.  0 is below every key.
//
// k <= 64: a wave keeps its k best, sorted, one per lane, and streams over its part of the row: a key at
//   or below the k-th best is dropped by one comparison, the few others wait in LDS until 64 of them
//   are sorted and merged into the list at once.  Four waves per workgroup, as many workgroups per row
//   as fill the chip; a second launch merges their lists.
// k > 64: a workgroup holds a tile of 8192 keys in registers, finds the tile's k-th largest by a radix
//   descent over LDS histograms (2048 bins a digit) and keeps the k keys at or above it; the kept
//   keys of all tiles are the next, 8192 / k times shorter, row.  The last level takes up to 16384 keys
//   in one workgroup and sorts.
#include "alsmi_common.h"
#include "elem.h"

#include <algorithm>
#include <type_traits>

namespace alsmi {

constexpr int TR_MAX_K = 1024;
constexpr int TR_LIST = 64;         // the longest list one wave keeps
constexpr int TR_CHUNK = 1024;      // keys a wave looks at per turn, 16 per lane
constexpr int TR_PART = 4 * TR_CHUNK;
constexpr int TR_THREADS = 512;     // k > 64: threads and keys per workgroup
constexpr int TR_TILE = 8192;
constexpr int TR_LAST = 16384;      // and of the last level's 1024 threads

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
    static __device__ __forceinline__ T score(type k) {
        const unsigned i = (unsigned)(k >> 32);
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
    static __device__ __forceinline__ unsigned short bits(type k) {
        const unsigned i = (unsigned)(k >> 32);
        return (unsigned short)((i & 0x8000u) ? (i & 0x7fffu) : ~i);
    }
};
template <>
struct RowKey<_Float16> : RowKey16 {
    static __device__ __forceinline__ image_t image(_Float16 s) {
        return RowKey16::image(__builtin_bit_cast(unsigned short, s));
    }
    static __device__ __forceinline__ _Float16 score(type k) {
        return __builtin_bit_cast(_Float16, bits(k));
    }
};
template <>
struct RowKey<__bf16> : RowKey16 {
    static __device__ __forceinline__ image_t image(__bf16 s) {
        return RowKey16::image(__builtin_bit_cast(unsigned short, s));
    }
    static __device__ __forceinline__ __bf16 score(type k) { return __builtin_bit_cast(__bf16, bits(k)); }
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
    static __device__ __forceinline__ double score(type k) {
        const unsigned long long i = (unsigned long long)(k >> 32);
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
        if (!SHORT) fetch(at + 4 * TR_CHUNK);  // (on its way while this chunk is looked at)
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
        scores_out[row * k + lane] = RowKey<T>::score(list);
    }
}

// ---- k > 64 --------------------------------------------------------------------------------------
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
// registers, all different but for zeros), by digits of 11 bits from the top; 0 if there are no k
// keys above it.  A pass costs its atomics and two barriers: every wave reads the whole histogram
// and finds the digit by itself (one wave, or sums by thread and prefix sums over the workgroup,
// with more barriers, took longer), and the other of two histograms is cleared meanwhile.
template <typename K, int THREADS, int E>
__device__ __forceinline__ K kth_key(const K (&key)[E], int k, int bits) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    constexpr int DIGIT = 11, BINS = 1 << DIGIT, LANE_BINS = BINS / 64;
    __shared__ u32x4 hist4[2][BINS / 4];
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
            if ((key[j] & upper) != prefix) continue;
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
        unsigned long long found = __ballot(upto >= want);  // (never 0: zeros are counted too)
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

// One tile of a row; SORT: the only tile of its row, whose k best are sorted and written out.
template <typename T, bool FROM_KEYS, bool SORT, int THREADS, int E>
__global__ __launch_bounds__(THREADS) void topk_tile_kernel(KeySource<T, FROM_KEYS> src, int k,
                                                            int index_bits, unsigned tiles,
                                                            typename RowKey<T>::type *__restrict__ kept,
                                                            int32_t *__restrict__ items_out,
                                                            T *__restrict__ scores_out) {
    typedef typename RowKey<T>::type key_t;
    constexpr int VEC = FROM_KEYS ? 16 / (int)sizeof(key_t) : 16 / (int)sizeof(T);
    static_assert(!SORT || THREADS == TR_MAX_K, "one key per thread to sort");
    __shared__ key_t sel[SORT ? TR_MAX_K : 1];
    __shared__ int n_kept;
    const int tid = threadIdx.x, lane = tid & 63;
    const unsigned r32 = blockIdx.x / tiles;
    const int64_t row = r32;
    const unsigned tile = blockIdx.x - r32 * tiles;
    const int64_t first = (int64_t)tile * (THREADS * E);
    key_t key[E];
#pragma unroll
    for (int j = 0; j < E; j += VEC) {
        typedef KeySource<T, FROM_KEYS> source;
        typename source::raw_t raw[VEC];
        const int64_t at = first + j * THREADS + tid * VEC;
        source::load(raw, src.data + row * src.ld, at, src.n);
#pragma unroll
        for (int i = 0; i < VEC; ++i) key[j + i] = source::key(raw[i], at + i, src.n);
    }
    if (tid == 0) n_kept = 0;
    key_t floor_key = 1;
    if (src.n - first > k) {
        // without the bits between image and index, which are ones in every key
        const unsigned index_mask = 0xffffffffu >> (32 - index_bits);
        auto without = [&](key_t x) { return ((x >> 32) << index_bits) | ((unsigned)x & index_mask); };
        key_t dense[E];
#pragma unroll
        for (int j = 0; j < E; ++j) dense[j] = without(key[j]);
        const key_t kth =
            kth_key<key_t, THREADS, E>(dense, k, RowKey<T>::BITS - 32 + index_bits);
        if (kth != 0)
            floor_key = ((kth >> index_bits) << 32) | (unsigned)~index_mask | ((unsigned)kth & index_mask);
    }
    __syncthreads();
    key_t *dst = SORT ? sel : kept + (row * tiles + tile) * k;
    unsigned mine_kept = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) mine_kept += key[j] >= floor_key;
    const unsigned upto = wave_prefix(mine_kept);
    int place = 0;
    if (lane == 63) place = atomicAdd(&n_kept, (int)upto);
    place = __builtin_amdgcn_readlane(place, 63) + (int)(upto - mine_kept);
#pragma unroll
    for (int j = 0; j < E; ++j)
        if (key[j] >= floor_key) dst[place++] = key[j];
    __syncthreads();
    const int have = n_kept;
    if constexpr (!SORT) {
        for (int i = have + tid; i < k; i += THREADS) dst[i] = 0;
    } else {
        // one key per thread: sorted by wave, then runs of 64, 128, ... meet the mirror image of the next
        // run; steps within a wave go through the lanes, the others through LDS
        key_t mine = wave_sort(tid < have ? sel[tid] : (key_t)0, lane);
        for (int size = 128; size < 2 * k; size <<= 1) {  // (runs behind the k-th key hold zeros)
            int mask = size - 1;
            for (int top = size >> 1; top >= 64; top >>= 1) {
                __syncthreads();
                sel[tid] = mine;
                __syncthreads();
                const key_t o = sel[tid ^ mask];
                mine = (o > mine) != ((tid & top) != 0) ? o : mine;
                mask = top >> 1;
            }
            mine = wave_merge(mine, lane);
        }
        if (tid < k) {
            items_out[row * k + tid] = (int32_t)~(unsigned)mine;
            scores_out[row * k + tid] = RowKey<T>::score(mine);
        }
    }
}

// ---- launches ------------------------------------------------------------------------------------
// k <= 64: workgroups per row, so that the launch has about 1024, at least 4096 keys each.
static int64_t list_parts(int64_t n_rows, int64_t n_items, int64_t &part_len) {
    const int64_t most = (n_items + TR_PART - 1) / TR_PART;
    int64_t parts = 1024 / n_rows;
    parts = parts < 1 ? 1 : (parts > most ? most : parts);
    part_len = ((n_items + parts - 1) / parts + TR_PART - 1) / TR_PART * TR_PART;
    return (n_items + part_len - 1) / part_len;
}
static int64_t tiles_of(int64_t n) { return (n + TR_TILE - 1) / TR_TILE; }
// Rows that are worked on at once: a launch has fewer than 2^32 threads.
static int64_t batch_rows(int64_t n_items, int k) {
    return k <= TR_LIST ? (int64_t)1 << 23 : std::max<int64_t>(1, ((int64_t)1 << 21) / tiles_of(n_items));
}

template <typename T>
static int run_lists(int64_t n_rows, const KeySource<T, false> &src, int k, int32_t *items_out,
                     T *scores_out, typename RowKey<T>::type *kept, hipStream_t st) {
    typedef typename RowKey<T>::type key_t;
    if (src.n <= TR_CHUNK) {
        hipLaunchKernelGGL((topk_list_kernel<T, false, true>), dim3((unsigned)((n_rows + 3) / 4)), dim3(256),
                           0, st, src, n_rows, k, 1u, src.n, (key_t *)nullptr, items_out, scores_out);
        ALSMI_HIP_CHECK(hipGetLastError());
        return ALSMI_OK;
    }
    int64_t part_len = 0;
    const int64_t parts = list_parts(n_rows, src.n, part_len);
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

template <typename T>
static int run_tiles(int64_t n_rows, const KeySource<T, false> &src, int k, int32_t *items_out,
                     T *scores_out, typename RowKey<T>::type *kept, hipStream_t st) {
    typedef typename RowKey<T>::type key_t;
    const dim3 last_grid((unsigned)n_rows), last_block(TR_MAX_K);
    int index_bits = 1;
    while (index_bits < 31 && (src.n - 1) >> index_bits) ++index_bits;
    if (src.n <= TR_LAST) {
        hipLaunchKernelGGL((topk_tile_kernel<T, false, true, TR_MAX_K, TR_LAST / TR_MAX_K>), last_grid,
                           last_block, 0, st, src, k, index_bits, 1u, (key_t *)nullptr, items_out, scores_out);
        ALSMI_HIP_CHECK(hipGetLastError());
        return ALSMI_OK;
    }
    int64_t tiles = tiles_of(src.n);
    hipLaunchKernelGGL((topk_tile_kernel<T, false, false, TR_THREADS, TR_TILE / TR_THREADS>),
                       dim3((unsigned)(tiles * n_rows)), dim3(TR_THREADS), 0, st, src, k, index_bits,
                       (unsigned)tiles, kept, (int32_t *)nullptr, (T *)nullptr);
    ALSMI_HIP_CHECK(hipGetLastError());
    // the levels alternate between the two parts of the workspace
    key_t *from = kept, *to = kept + n_rows * tiles * k;
    int64_t n = tiles * k;
    while (n > TR_LAST) {
        tiles = tiles_of(n);
        const KeySource<T, true> left = {from, n, n};
        hipLaunchKernelGGL((topk_tile_kernel<T, true, false, TR_THREADS, TR_TILE / TR_THREADS>),
                           dim3((unsigned)(tiles * n_rows)), dim3(TR_THREADS), 0, st, left, k, index_bits,
                           (unsigned)tiles, to, (int32_t *)nullptr, (T *)nullptr);
        ALSMI_HIP_CHECK(hipGetLastError());
        key_t *t = from;
        from = to;
        to = t;
        n = tiles * k;
    }
    const KeySource<T, true> left = {from, n, n};
    hipLaunchKernelGGL((topk_tile_kernel<T, true, true, TR_MAX_K, TR_LAST / TR_MAX_K>), last_grid,
                       last_block, 0, st, left, k, index_bits, 1u, (key_t *)nullptr, items_out, scores_out);
    ALSMI_HIP_CHECK(hipGetLastError());
    return ALSMI_OK;
}

template <typename T>
static int run_topk_rows(int64_t n_rows, int64_t n_items, const void *scores, int64_t ld, int k,
                         int32_t *items_out, void *scores_out, void *workspace, hipStream_t st) {
    typedef typename RowKey<T>::type key_t;
    T *so = static_cast<T *>(scores_out);
    key_t *kept = static_cast<key_t *>(workspace);
    const int64_t most = batch_rows(n_items, k);  // (the workspace serves one batch after the other)
    for (int64_t lo = 0; lo < n_rows; lo += most) {
        const int64_t rows = std::min(n_rows - lo, most);
        const KeySource<T, false> src = {static_cast<const T *>(scores) + lo * ld, ld, n_items};
        const int status = k <= TR_LIST
                               ? run_lists<T>(rows, src, k, items_out + lo * k, so + lo * k, kept, st)
                               : run_tiles<T>(rows, src, k, items_out + lo * k, so + lo * k, kept, st);
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
    int64_t keys = 0;
    n_rows = std::min(n_rows, batch_rows(n_items, k));
    if (k <= TR_LIST) {
        int64_t part_len = 0;
        const int64_t parts = list_parts(n_rows, n_items, part_len);
        keys = parts > 1 ? parts * k : 0;
    } else if (n_items > TR_LAST) {
        const int64_t n = tiles_of(n_items) * k;
        keys = n + (n > TR_LAST ? tiles_of(n) * k : 0);
    }
    return (size_t)n_rows * (size_t)keys * (dtype == ALSMI_F64 ? 16 : 8) + 16;
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
