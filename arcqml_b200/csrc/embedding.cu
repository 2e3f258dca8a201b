// embedding.cu — rows of a table looked up by index (token embeddings, or states normalised from trained
// amplitudes), and that lookup's gradient by sorted indices.
//
//   lookup    out[i] = s t[x_i], or s t[x_i] / |t[x_i]|
//   gradient  G_v = s sum of g_i over the places i with x_i = v, in the places' order; for normalised rows
//             (G_v - u <u, G_v>) / |t_v| with u = t_v / |t_v|: every place of a row has the same u, so the
//             sum is formed first and taken through the norm once
//
// Both move each number once and do next to nothing with it: the latency of index, row and store bounds them
// at real sizes (at 60 to 70 % of the copy rate), launches at small ones. The gradient's places are sorted by their row first (a stable radix sort, so that a row's
// places stay in order and equal inputs give equal bits without atomics on values); chunks of the sorted
// places are then summed side by side, whatever rows they belong to, so a row that most places point to
// costs no more than others; rows that cross chunks are put together from the chunks' partial sums.
//
//   k_lookup, k_lookup_row, k_row_squares   rows as they are; normalised in registers; in pieces
//   k_direct                                the gradient of few places, in one launch
//   k_sort_cluster                          up to 131072 places sorted, the output cleared beside that
//   k_count_digits, k_prefix_counts,
//   k_sort_pass, k_zero_rows                more places
//   k_sum_chunks, k_join_chunks, k_project  sums of chunks, rows across them, the norm
//
// Measured on a B200 (copy rate 6543 GB/s): 65,536 bf16 rows of 2 KB at random, scaled, 36 us a call (4.6 TB/s of
// algorithmic bytes); 1024 normalised rows of 16 KB 8.9 us in the kernel, 11 us a call (the host's time);
// the gradient of 131,071 bf16 places in 50,021 rows of 2 KB 120 us a call: 32 us the sort, 66 us the sums
// (4.1 TB/s), 19 us the rows across chunks; of 1024 places in 509 normalised rows of 16 KB 13.5 us a call.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <sstream>
#include <string>
#include <tuple>
#include <type_traits>

#include "elements.cuh"
#include "embedding.h"
#include "launch.h"
#include "profile.h"

namespace cg = cooperative_groups;

namespace arcqml {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kAbsent = 0xffffffffu; // the key of a place that counts nowhere

// Indices as they lie in memory.
struct Indices {
    const void *at;
    uint64_t rows;
    int64_t padding;
    uint32_t wide; // 8 bytes each
    __device__ __forceinline__ int64_t operator[](uint64_t i) const {
        return wide ? __ldg(static_cast<const long long *>(at) + i)
                    : int64_t(__ldg(static_cast<const int *>(at) + i));
    }
    __device__ __forceinline__ bool inside(int64_t x) const { return uint64_t(x) < rows; }
    __device__ __forceinline__ bool is_padding(int64_t x) const { return padding >= 0 && x == padding; }
};

struct Lookup {
    const char *table;
    char *out;
    Indices index;
    uint64_t places, stride, row_bytes; // stride: bytes between the table's rows
    double scale;
    // of normalised rows in pieces: sums of squares, `pieces` for each place; of f64, negative ones were formed of
    // numbers 2^-n times as large, n lies `places * pieces` behind them
    const double *squares;
    uint32_t vectors;      // of a row
    uint32_t lanes;        // a power of two: threads that share a tile
    uint32_t tiles, pieces;
};

constexpr uint32_t kTileVectors = 4;   // vectors of a tile for each of its threads
constexpr uint32_t kRowVectors = 8;    // of a normalised row that its threads hold in registers
constexpr uint32_t kPieceVectors = 2048;

// ------------------------------------------------------------------ lookup

constexpr uint32_t kNotANumber = 0x7fffffff; // as every word of a vector: NaN in each type

// Squares of f64 leave its range long before the numbers do. A row whose sum of squares is near the range's ends
// (what is lost below 2^-900 is 2^-174 of it or less) is gone through again with numbers 2^-n times as large, n the
// exponent of its largest one; squares of the other types stay far inside. A NaN or an infinity stays what it is.
template <class W> __device__ __forceinline__ bool out_of_range(double squares) {
    return sizeof(W) == 8 && (squares < 0x1p-900 || squares > 0x1p900);
}
__device__ __forceinline__ int power_of(double largest) {
    return largest > 0.0 && largest < INFINITY ? ilogb(largest) : 0;
}
// x 2^-power for powers of finite numbers, by two factors: one would leave the range.
__device__ __forceinline__ double lowered(double x, int power) {
    const int half = power / 2, rest = power - half;
    return x * __hiloint2double((1023 - half) << 20, 0) * __hiloint2double((1023 - rest) << 20, 0);
}
// Numbers of a vector 2^-power times as large.
template <class T, int N> __device__ __forceinline__ void rescale(Packed<T, N> &v, int power) {
    if constexpr (sizeof(T) == 8) {
        double x[N];
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = lowered(v.wide(e), power);
        v.pack(x);
    }
}

// Rows in tiles of 4 vectors a thread, a tile taken by `lanes` threads: 2 KB a warp, four loads in flight for
// each thread. 34 us for 65,536 rows of 2 KB (243 MB, 112 of them from and to DRAM, the rest L2's) at half of what
// memory and SMs take: a warp lives for one index -> row -> store, and waits for most of that.
template <uint32_t DT, int N>
__global__ void __launch_bounds__(kThreads) k_lookup(const __grid_constant__ Lookup a) {
    using T = Element<DT>;
    using W = WideElement<DT>;
    const uint64_t unit = (uint64_t(blockIdx.x) * kThreads + threadIdx.x) / a.lanes;
    const uint32_t lane = threadIdx.x & (a.lanes - 1);
    const uint64_t place = unit / a.tiles;
    if (place >= a.places) return;
    const uint32_t first = uint32_t(unit % a.tiles) * a.lanes * kTileVectors + lane;
    const int64_t row = a.index[place];
    const bool inside = a.index.inside(row), padding = a.index.is_padding(row);
    const char *from = a.table + (inside ? uint64_t(row) : 0) * a.stride;
    char *to = a.out + place * a.row_bytes;
    Packed<T, N> v[kTileVectors];
#pragma unroll
    for (uint32_t j = 0; j < kTileVectors; ++j) {
        const uint32_t k = first + j * a.lanes;
        if (inside && k < a.vectors) v[j].load(from + uint64_t(k) * Packed<T, N>::BYTES);
    }
    double factor = a.scale;
    if (a.squares) {
        double sum = 0.0;
        if (inside && !padding) {
            const double *squares = a.squares + place * a.pieces, *powers = squares + a.places * a.pieces;
            bool apart = false;
            for (uint32_t p = 0; p < a.pieces; ++p) {
                sum += squares[p];
                apart = apart || squares[p] < 0.0;
            }
            if (sizeof(W) == 8 && apart) { // pieces of different powers: all by the largest one's
                int power = -4096;
#pragma unroll 1
                for (uint32_t p = 0; p < a.pieces; ++p)
                    if (squares[p] != 0.0) power = max(power, squares[p] < 0.0 ? int(powers[p]) : 0);
                sum = 0.0;
#pragma unroll 1
                for (uint32_t p = 0; p < a.pieces; ++p) {
                    const int below = power - (squares[p] < 0.0 ? int(powers[p]) : 0);
                    // (2^-1200 times as large, a piece is nothing beside the largest)
                    if (below < 600) sum += lowered(fabs(squares[p]), 2 * below);
                }
#pragma unroll
                for (uint32_t j = 0; j < kTileVectors; ++j) rescale(v[j], power);
            }
        }
        factor = sum == 0.0 ? 0.0 : a.scale / sqrt(sum);
    }
    const bool plain = !a.squares && factor == 1.0; // the rows as they are
#pragma unroll
    for (uint32_t j = 0; j < kTileVectors; ++j) {
        const uint32_t k = first + j * a.lanes;
        if (k >= a.vectors) continue;
        Packed<T, N> y = v[j];
        if (padding || !inside) {
            y.fill(padding ? 0 : kNotANumber);
        } else if (!plain) {
            W x[N];
#pragma unroll
            for (int e = 0; e < N; ++e)
                x[e] = a.squares ? W(double(v[j].wide(e)) * factor) : v[j].wide(e) * W(factor);
            y.pack(x);
        }
        y.store(to + uint64_t(k) * Packed<T, N>::BYTES);
    }
}

// The sum over `lanes` threads (up to a block's), the same in each of them.
template <bool BLOCK> __device__ __forceinline__ double sum_over(double v, uint32_t lanes) {
    const uint32_t within = BLOCK ? 32 : lanes;
    for (uint32_t o = within / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, int(o));
    if constexpr (BLOCK) {
        __shared__ double part[kThreads / 32];
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.0;
        for (int w = 0; w < kThreads / 32; ++w) v += part[w];
    }
    return v;
}

// The largest over `lanes` threads.
template <bool BLOCK> __device__ __forceinline__ double largest_over(double v, uint32_t lanes) {
    const uint32_t within = BLOCK ? 32 : lanes;
    for (uint32_t o = within / 2; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, int(o)));
    if constexpr (BLOCK) {
        __shared__ double part[kThreads / 32];
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
        __syncthreads(); // (behind the last use of sum_over's shared memory, too)
        v = 0.0;
        for (int w = 0; w < kThreads / 32; ++w) v = fmax(v, part[w]);
    }
    return v;
}

// Normalised rows that their threads hold (read once): `lanes` threads of a warp up to 4 KB a row, or a block
// up to 32 KB, for each place. 8.9 us for 1024 rows of 16 KB from and to HBM: latency of one round.
template <uint32_t DT, int N, bool BLOCK>
__global__ void __launch_bounds__(kThreads) k_lookup_row(const __grid_constant__ Lookup a) {
    using T = Element<DT>;
    using W = WideElement<DT>;
    const uint32_t lanes = BLOCK ? kThreads : a.lanes;
    const uint64_t place = BLOCK ? blockIdx.x : (uint64_t(blockIdx.x) * kThreads + threadIdx.x) / lanes;
    const uint32_t lane = threadIdx.x & (lanes - 1);
    const bool on = place < a.places;
    const int64_t row = on ? a.index[place] : -1;
    const bool inside = a.index.inside(row), padding = a.index.is_padding(row);
    const char *from = a.table + (inside ? uint64_t(row) : 0) * a.stride;
    Packed<T, N> v[kRowVectors];
#pragma unroll
    for (uint32_t j = 0; j < kRowVectors; ++j) {
        const uint32_t k = lane + j * lanes;
        if (inside && !padding && k < a.vectors) v[j].load(from + uint64_t(k) * Packed<T, N>::BYTES);
        else
#pragma unroll
            for (int i = 0; i < Packed<T, N>::WORDS; ++i) v[j].w[i] = 0;
    }
    double sum = 0.0;
#pragma unroll
    for (uint32_t j = 0; j < kRowVectors; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const double x = v[j].wide(e);
            sum = fma(x, x, sum);
        }
    sum = sum_over<BLOCK>(sum, lanes);
    const bool far = inside && !padding && out_of_range<W>(sum);
    if (sizeof(W) == 8 && __any_sync(0xffffffffu, far)) { // one of the warp's rows; the block's one
        double largest = 0.0;
#pragma unroll
        for (uint32_t j = 0; j < kRowVectors; ++j)
#pragma unroll
            for (int e = 0; e < N; ++e) largest = fmax(largest, fabs(double(v[j].wide(e))));
        largest = largest_over<BLOCK>(largest, lanes);
        const int power = far ? power_of(largest) : 0;
        double again = 0.0;
#pragma unroll
        for (uint32_t j = 0; j < kRowVectors; ++j) {
            rescale(v[j], power);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const double x = v[j].wide(e);
                again = fma(x, x, again);
            }
        }
        sum = sum_over<BLOCK>(again, lanes); // a row in the range has the same one again
    }
    const double factor = sum == 0.0 ? 0.0 : a.scale / sqrt(sum);
    char *to = a.out + place * a.row_bytes;
#pragma unroll
    for (uint32_t j = 0; j < kRowVectors; ++j) {
        const uint32_t k = lane + j * lanes;
        if (!on || k >= a.vectors) continue;
        Packed<T, N> y;
        if (padding || !inside) {
            y.fill(padding ? 0 : kNotANumber);
        } else {
            W x[N];
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = W(double(v[j].wide(e)) * factor);
            y.pack(x);
        }
        y.store(to + uint64_t(k) * Packed<T, N>::BYTES);
    }
}

// Squares of one piece of the row of one place: a block each.
template <uint32_t DT, int N>
__global__ void __launch_bounds__(kThreads) k_row_squares(const __grid_constant__ Lookup a, double *squares) {
    using T = Element<DT>;
    const uint64_t place = blockIdx.x / a.pieces;
    const uint32_t piece = blockIdx.x % a.pieces;
    const int64_t row = a.index[place];
    const char *from = a.table + (a.index.inside(row) ? uint64_t(row) : 0) * a.stride;
    const uint32_t first = piece * kPieceVectors;
    const uint32_t end = a.index.inside(row) && !a.index.is_padding(row) ? min(a.vectors, first + kPieceVectors) : first;
    const auto over_row = [&](auto &&use) {
#pragma unroll 8
        for (uint32_t k = first + threadIdx.x; k < end; k += kThreads) {
            Packed<T, N> v;
            v.load(from + uint64_t(k) * Packed<T, N>::BYTES);
#pragma unroll
            for (int e = 0; e < N; ++e) use(v.wide(e));
        }
    };
    double sum = 0.0;
    over_row([&](double x) { sum = fma(x, x, sum); });
    sum = sum_over<true>(sum, kThreads);
    const uint64_t at = place * a.pieces + piece;
    if (end > first && out_of_range<WideElement<DT>>(sum)) { // the same in the whole block
        double largest = 0.0;
        over_row([&](double x) { largest = fmax(largest, fabs(x)); });
        const int power = power_of(largest_over<true>(largest, kThreads));
        if (power) {
            sum = 0.0;
            over_row([&](double x) {
                x = lowered(x, power);
                sum = fma(x, x, sum);
            });
            sum = -sum_over<true>(sum, kThreads);
            if (threadIdx.x == 0) squares[a.places * a.pieces + at] = power;
        }
    }
    if (threadIdx.x == 0) squares[at] = sum;
}

// ------------------------------------------------------------------ sorting the places by their rows

// Keys are rows; places that count nowhere have the key kAbsent and end up last. A pass takes up to 9
// bits; blocks of 2048 keys are ranked by their warps in the order of the places.
constexpr uint32_t kBins = 512, kSortKeys = 2048, kKeysPerThread = kSortKeys / kThreads;
constexpr uint32_t kWarps = kThreads / 32;

struct Sort {
    Indices index;
    const uint2 *from; // keys with their places; null in the first pass, which reads the indices
    uint2 *out;
    uint32_t *counts; // [blocks][kBins] of this pass, as prefixes over the blocks if `totals` is not null
    uint32_t *totals; // [kBins]
    uint32_t *next;   // counts of the next pass, zero so far; null in the last one
    uint32_t places, blocks, shift, next_shift, bits;
};

__device__ __forceinline__ uint32_t key_at(const Indices &x, uint64_t i) {
    const int64_t v = x[i];
    return x.inside(v) && !x.is_padding(v) ? uint32_t(v) : kAbsent;
}
__device__ __forceinline__ uint32_t digit_of(uint32_t key, uint32_t shift, uint32_t bits) {
    return key >> shift & ((1u << bits) - 1);
}

// The lanes whose digit is this lane's, a ballot for each bit (a match instruction takes about 100 cycles: the
// sort of 131071 places took 40 us with it).
__device__ __forceinline__ uint32_t lanes_alike(uint32_t digit, uint32_t bits) {
    uint32_t same = 0xffffffffu;
#pragma unroll
    for (uint32_t b = 0; b < 9; ++b) {
        if (b >= bits) break;
        const uint32_t all = uint32_t(int32_t(digit << (31 - b)) >> 31); // the bit, everywhere
        same &= ~(__ballot_sync(0xffffffffu, all != 0) ^ all);
    }
    return same;
}

// The first pass's counts; clears those of the passes behind it (`clear` words at s.next).
__global__ void __launch_bounds__(kThreads) k_count_digits(const __grid_constant__ Sort s, uint64_t clear) {
    __shared__ uint32_t bins[kBins];
    cudaTriggerProgrammaticLaunchCompletion();
    for (uint32_t b = threadIdx.x; b < kBins; b += kThreads) bins[b] = 0;
    for (uint64_t i = uint64_t(blockIdx.x) * kThreads + threadIdx.x; i < clear; i += uint64_t(gridDim.x) * kThreads)
        s.next[i] = 0;
    __syncthreads();
    const uint32_t end = uint32_t(min(uint64_t(s.places), (uint64_t(blockIdx.x) + 1) * kSortKeys));
    for (uint32_t i = blockIdx.x * kSortKeys + threadIdx.x; i < end; i += kThreads)
        atomicAdd(&bins[digit_of(key_at(s.index, i), s.shift, s.bits)], 1u);
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < kBins; b += kThreads) s.counts[uint64_t(blockIdx.x) * kBins + b] = bins[b];
}

// For many blocks: counts -> the number of the digit's keys in earlier blocks, and the digits' totals.
// A block takes 32 digits, 32 threads each.
__global__ void __launch_bounds__(1024) k_prefix_counts(uint32_t *counts, uint32_t *totals, uint32_t blocks) {
    __shared__ uint32_t part[32][33];
    cudaTriggerProgrammaticLaunchCompletion();
    cudaGridDependencySynchronize();
    const uint32_t digit = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
    const uint32_t each = (blocks + 31) / 32, lo = slice * each, hi = min(blocks, lo + each);
    uint32_t sum = 0;
    for (uint32_t b = lo; b < hi; ++b) sum += counts[uint64_t(b) * kBins + digit];
    part[slice][threadIdx.x & 31] = sum;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (uint32_t i = 0; i < 32; ++i) {
        if (i == slice) before = all;
        all += part[i][threadIdx.x & 31];
    }
    for (uint32_t b = lo; b < hi; ++b) {
        const uint32_t c = counts[uint64_t(b) * kBins + digit];
        counts[uint64_t(b) * kBins + digit] = before;
        before += c;
    }
    if (slice == 0) totals[digit] = all;
}

__global__ void __launch_bounds__(kThreads) k_sort_pass(const __grid_constant__ Sort s) {
    __shared__ uint32_t hist[kWarps][kBins];
    __shared__ uint32_t base[kBins];
    __shared__ uint32_t warp_sum[kWarps];
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
    cudaTriggerProgrammaticLaunchCompletion();
    for (uint32_t b = t; b < kWarps * kBins; b += kThreads) (&hist[0][0])[b] = 0;
    __syncthreads();
    cudaGridDependencySynchronize();
    uint32_t key[kKeysPerThread], place[kKeysPerThread], rank[kKeysPerThread];
    const uint32_t first = blockIdx.x * kSortKeys + warp * (kSortKeys / kWarps) + lane;
#pragma unroll
    for (uint32_t j = 0; j < kKeysPerThread; ++j) {
        const uint32_t i = first + j * 32;
        place[j] = i;
        key[j] = kAbsent;
        if (i < s.places && s.from) key[j] = s.from[i].x, place[j] = s.from[i].y;
        else if (i < s.places) key[j] = key_at(s.index, i);
    }
#pragma unroll
    for (uint32_t j = 0; j < kKeysPerThread; ++j) {
        const bool on = first + j * 32 < s.places; // the warp's first lanes, all of it but at the end
        const uint32_t d = digit_of(key[j], s.shift, s.bits);
        const uint32_t same = lanes_alike(d, s.bits) & __ballot_sync(0xffffffffu, on);
        const uint32_t before = __popc(same & ((1u << lane) - 1));
        if (on) rank[j] = hist[warp][d] + before;
        __syncwarp();
        if (on && before == 0) hist[warp][d] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    // each thread: two neighbouring digits
    uint32_t all[2], mine[2];
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
        const uint32_t d = 2 * t + h;
        uint32_t sum = 0;
        for (uint32_t w = 0; w < kWarps; ++w) {
            const uint32_t c = hist[w][d];
            hist[w][d] = sum;
            sum += c;
        }
        all[h] = mine[h] = 0;
        if (s.totals) {
            all[h] = s.totals[d];
            mine[h] = s.counts[uint64_t(blockIdx.x) * kBins + d];
        }
    }
    if (!s.totals) {
#pragma unroll 8
        for (uint32_t b = 0; b < s.blocks; ++b) {
            const uint2 c = *reinterpret_cast<const uint2 *>(s.counts + uint64_t(b) * kBins + 2 * t);
            if (b < blockIdx.x) {
                mine[0] += c.x;
                mine[1] += c.y;
            }
            all[0] += c.x;
            all[1] += c.y;
        }
    }
    uint32_t sum = all[0] + all[1], scan = sum;
    for (uint32_t o = 1; o < 32; o *= 2) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += up;
    }
    if (lane == 31) warp_sum[warp] = scan;
    __syncthreads();
    uint32_t before = scan - sum;
    for (uint32_t w = 0; w < warp; ++w) before += warp_sum[w];
    base[2 * t] = before + mine[0];
    base[2 * t + 1] = before + all[0] + mine[1];
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < kKeysPerThread; ++j) {
        const uint32_t i = first + j * 32;
        if (i >= s.places) continue;
        const uint32_t d = digit_of(key[j], s.shift, s.bits);
        const uint32_t to = base[d] + hist[warp][d] + rank[j];
        s.out[to] = make_uint2(key[j], place[j]);
        if (s.next) atomicAdd(&s.next[uint64_t(to / kSortKeys) * kBins + digit_of(key[j], s.next_shift, s.bits)], 1u);
    }
}

// Up to 16 blocks of a cluster sort up to 131072 keys in one launch; their counts go through distributed
// shared memory, the keys through L2 (stores into other blocks' shared memory took no less). A pass takes about
// 25,000 cycles, 8,000 of them for the ballots of the ranks. The other clusters of the launch clear the output
// meanwhile: most of its rows are often absent, and it is written twice only where a row is present.
// Each thread has 1, 2, 4 or 8 keys: as few as 16 blocks leave it, since ranking takes 1000 cycles for each
// (8192 places: 25 us in one block, see the call's times for more).
constexpr uint32_t kClusterThreads = 1024, kMostPerThread = 8;
constexpr uint32_t kClusterWarps = kClusterThreads / 32, kMostCluster = 16;

struct ClusterSort {
    Indices index;
    uint2 *out[2]; // the sorted keys, and room for a pass before the last
    char *clear;
    uint64_t clear_bytes;
    uint32_t places, passes, bits;
};
struct ClusterShared {
    uint16_t hist[kClusterWarps][kBins];
    uint32_t total[2][kBins]; // of this block, by parity of the pass
    uint32_t base[kBins]; // where this block's keys of a digit begin
    uint32_t warp_sum[kClusterWarps];
};

__device__ __forceinline__ void clear_share(char *to, uint64_t bytes, uint64_t thread, uint64_t threads) {
    const uint64_t head = min(bytes, uint64_t(-reinterpret_cast<uintptr_t>(to) & 15)), body = (bytes - head) / 16;
    if (thread < head) to[thread] = 0;
    uint4 *v = reinterpret_cast<uint4 *>(to + head);
    for (uint64_t i = thread; i < body; i += threads) v[i] = make_uint4(0, 0, 0, 0);
    const uint64_t tail = head + body * 16;
    if (thread < bytes - tail) to[tail + thread] = 0;
}

template <uint32_t PER_THREAD>
__global__ void __launch_bounds__(kClusterThreads, 1) k_sort_cluster(const __grid_constant__ ClusterSort s) {
    constexpr uint32_t KEYS = PER_THREAD * kClusterThreads;
    extern __shared__ char raw[];
    ClusterShared &sh = *reinterpret_cast<ClusterShared *>(raw);
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t size = cluster.num_blocks(), me = cluster.block_rank();
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
    cudaTriggerProgrammaticLaunchCompletion();
    if (blockIdx.x >= size) {
        clear_share(s.clear, s.clear_bytes, uint64_t(blockIdx.x - size) * kClusterThreads + t,
                    uint64_t(gridDim.x - size) * kClusterThreads);
        return;
    }
    for (uint32_t p = 0; p < s.passes; ++p) {
        const uint32_t shift = p * s.bits, parity = p & 1;
        const bool last = p + 1 == s.passes;
        // the last pass writes out[0]
        uint2 *to = s.out[(s.passes - 1 - p) & 1];
        const uint2 *from = s.out[(s.passes - p) & 1];
        for (uint32_t b = t; b < kClusterWarps * kBins / 2; b += kClusterThreads)
            reinterpret_cast<uint32_t *>(&sh.hist[0][0])[b] = 0;
        __syncthreads();
        uint2 key[PER_THREAD];
        uint32_t rank[PER_THREAD];
        const uint32_t first = me * KEYS + warp * (KEYS / kClusterWarps) + lane;
#pragma unroll
        for (uint32_t j = 0; j < PER_THREAD; ++j) {
            // keys behind the last place sort behind all others and stay where they are
            const uint32_t i = first + j * 32;
            key[j] = make_uint2(kAbsent, i);
            if (i < s.places) {
                if (p) key[j] = __ldcg(from + i);
                else key[j].x = key_at(s.index, i);
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < PER_THREAD; ++j) {
            const uint32_t d = digit_of(key[j].x, shift, s.bits), same = lanes_alike(d, s.bits);
            const uint32_t before = __popc(same & ((1u << lane) - 1));
            rank[j] = sh.hist[warp][d] + before;
            __syncwarp();
            if (before == 0) sh.hist[warp][d] = uint16_t(rank[j] + __popc(same));
            __syncwarp();
        }
        __syncthreads();
        if (t < kBins) { // a thread for each digit
            uint32_t sum = 0;
#pragma unroll 8
            for (uint32_t w = 0; w < kClusterWarps; ++w) {
                const uint32_t c = sh.hist[w][t];
                sh.hist[w][t] = uint16_t(sum);
                sum += c;
            }
            sh.total[parity][t] = sum;
        }
        cluster.sync();
        uint32_t all = 0, mine = 0;
        if (t < kBins) {
            for (uint32_t b = 0; b < size; ++b) {
                const uint32_t c = cluster.map_shared_rank(&sh, b)->total[parity][t];
                if (b < me) mine += c;
                all += c;
            }
        }
        uint32_t scan = all;
        for (uint32_t o = 1; o < 32; o *= 2) {
            const uint32_t up = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += up;
        }
        if (lane == 31) sh.warp_sum[warp] = scan;
        __syncthreads();
        if (t < kBins) {
            uint32_t before = scan - all + mine;
            for (uint32_t w = 0; w < warp; ++w) before += sh.warp_sum[w];
            sh.base[t] = before;
        }
        __syncthreads();
        // (the last pass: nobody reads this block's counts any more; it need not wait for its own stores)
        if (last) cluster.barrier_arrive();
#pragma unroll
        for (uint32_t j = 0; j < PER_THREAD; ++j) {
            const uint32_t d = digit_of(key[j].x, shift, s.bits);
            const uint32_t at = sh.base[d] + sh.hist[warp][d] + rank[j];
            if (at < s.places) to[at] = key[j];
        }
        if (last) {
            cluster.barrier_wait();
        } else {
            __threadfence();
            cluster.sync(); // the next pass's keys are there
        }
    }
}

// ------------------------------------------------------------------ sums of the rows' places

struct Sums {
    const char *gradient;
    char *out;
    const uint2 *sorted; // the rows with their places
    void *partial;             // [2 chunks][width] of the wide type: rows that cross chunks
    uint64_t stride;           // bytes between the gradient's rows
    uint64_t width, rows;
    double scale;
    uint32_t places, chunk, chunks;
    uint32_t vectors, lanes, tiles;
};

// Places at a time in flight for each thread.
constexpr uint32_t kAhead = 8;

template <class T, class O, class W, int N>
__device__ __forceinline__ void write_sum(const Sums &a, uint32_t row, uint32_t vector, const W (&sum)[N]) {
    constexpr int PART = sizeof(O) * N > 16 ? 16 / int(sizeof(O)) : N; // sums of 16-bit rows in 32 bits: two stores
    char *to = a.out + (uint64_t(row) * a.width + uint64_t(vector) * N) * sizeof(O);
#pragma unroll
    for (int p = 0; p < N; p += PART) {
        Packed<O, PART> v;
        W x[PART];
#pragma unroll
        for (int e = 0; e < PART; ++e) x[e] = sum[p + e] * W(a.scale);
        v.pack(x);
        v.store(to + p * sizeof(O));
    }
}

// One vector of a row for each thread, over the places of one chunk, eight of them in flight: what bounds it is
// the latency of rows at random (66 us for 131,071 rows of 2 KB, 4.1 TB/s; vectors through slots of shared
// memory by cp.async, 16 in flight, took 76 us; whole rows of 2 KB a warp 126 us, for want of registers). Three
// blocks an SM leave a thread 80 registers, and up to 80 bytes of what it holds are spilled (60 bytes for vectors
// of 8 bf16 numbers). A row that lies inside the chunk is done; the part of one that began earlier goes to
// partial 2c, of one that goes on to 2c + 1.
template <uint32_t DT, uint32_t OT, int N>
__global__ void __launch_bounds__(kThreads, 3) k_sum_chunks(const __grid_constant__ Sums a) {
    using T = Element<DT>;
    using O = Element<OT>;
    using W = WideElement<DT>;
    cudaTriggerProgrammaticLaunchCompletion();
    const uint64_t unit = (uint64_t(blockIdx.x) * kThreads + threadIdx.x) / a.lanes;
    const uint32_t c = uint32_t(unit / a.tiles);
    const uint32_t vector = uint32_t(unit % a.tiles) * a.lanes + (threadIdx.x & (a.lanes - 1));
    if (c >= a.chunks || vector >= a.vectors) return;
    cudaGridDependencySynchronize();
    const uint32_t i0 = c * a.chunk, i1 = min(a.places, i0 + a.chunk);
    uint32_t row = a.sorted[i0].x, begin = i0;
    if (row == kAbsent) return;
    W sum[N];
    const auto clear = [&] {
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = W(0);
    };
    clear();
    const auto flush = [&](uint32_t end) {
        const bool starts = begin > i0 || i0 == 0 || a.sorted[i0 - 1].x != row;
        const bool ends = end < i1 || i1 == a.places || a.sorted[i1].x != row;
        if (starts && ends) {
            write_sum<T, O, W, N>(a, row, vector, sum);
        } else {
            W *p = static_cast<W *>(a.partial) + (uint64_t(2) * c + (starts ? 1 : 0)) * a.width + uint64_t(vector) * N;
#pragma unroll
            for (int e = 0; e < N; ++e) p[e] = sum[e];
        }
    };
    const char *column = a.gradient + uint64_t(vector) * Packed<T, N>::BYTES;
    for (uint32_t i = i0; i < i1; i += kAhead) {
        Packed<T, N> v[kAhead];
        uint32_t key[kAhead];
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            const uint2 p = i + j < i1 ? a.sorted[i + j] : make_uint2(kAbsent, 0);
            key[j] = p.x;
            if (key[j] != kAbsent) v[j].load(column + uint64_t(p.y) * a.stride);
        }
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            if (key[j] != row) {
                if (row != kAbsent) flush(i + j);
                row = key[j];
                begin = i + j;
                clear();
            }
            if (key[j] == kAbsent) break;
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] += v[j].wide(e);
        }
        if (row == kAbsent) return;
    }
    flush(i1);
}

// The first place in the sorted keys that is not below `key`.
__device__ __forceinline__ uint32_t first_not_below(const uint2 *sorted, uint32_t n, uint32_t key) {
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (sorted[mid].x < key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// Rows that began in a chunk and went on: a block for each chunk and 32 vectors (19 us after 131,071 places, of
// which 8,400 belong to one row). Its warps add up an eighth
// of the row's partial sums each, in order, then the first one the eighths.
template <uint32_t DT, uint32_t OT, int N>
__global__ void __launch_bounds__(kThreads) k_join_chunks(const __grid_constant__ Sums a) {
    using T = Element<DT>;
    using O = Element<OT>;
    using W = WideElement<DT>;
    __shared__ W part[kWarps][32][N];
    const uint32_t groups = (a.vectors + 31) / 32, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t c = blockIdx.x / groups, vector = blockIdx.x % groups * 32 + lane;
    cudaTriggerProgrammaticLaunchCompletion();
    cudaGridDependencySynchronize();
    const uint32_t i0 = c * a.chunk, i1 = i0 + a.chunk, row = a.sorted[i1 - 1].x;
    if (row == kAbsent || a.sorted[i1].x != row) return;
    if (a.sorted[i0].x == row && i0 != 0 && a.sorted[i0 - 1].x == row) return; // it began earlier
    uint32_t last = c; // the chunk in which the row ends: the first one that does not end with it, or the last of all
    for (bool on = true; on;) {
        const uint32_t d = last + 1 + lane, end = (d + 1) * a.chunk;
        const bool goes_on = d + 1 < a.chunks && a.sorted[end - 1].x == row && a.sorted[end].x == row;
        const uint32_t stops = __ballot_sync(0xffffffffu, !goes_on);
        on = stops == 0;
        last += on ? 32 : __ffs(int(stops));
    }
    // the first partial is 2c + 1, the others 2d for d = c + 1 .. last
    const uint32_t count = last - c, each = (count + kWarps - 1) / kWarps, lo = c + 1 + warp * each, hi = min(last + 1, lo + each);
    W sum[N];
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] = W(0);
    const bool on = vector < a.vectors;
    const W *p = static_cast<const W *>(a.partial) + uint64_t(vector) * N;
    if (on && warp == 0)
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = p[(uint64_t(2) * c + 1) * a.width + e];
    if (on)
#pragma unroll 8
        for (uint32_t d = lo; d < hi; ++d)
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] += p[uint64_t(2) * d * a.width + e];
#pragma unroll
    for (int e = 0; e < N; ++e) part[warp][lane][e] = sum[e];
    __syncthreads();
    if (warp != 0 || !on) return;
    for (uint32_t w = 1; w < kWarps; ++w)
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += part[w][lane][e];
    write_sum<T, O, W, N>(a, row, vector, sum);
}

// Rows that no index points to: a warp looks at 32 rows.
template <uint32_t OT> __global__ void __launch_bounds__(kThreads) k_zero_rows(const __grid_constant__ Sums a) {
    using O = Element<OT>;
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t first = (uint64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * 32;
    cudaTriggerProgrammaticLaunchCompletion();
    if (first >= a.rows) return;
    cudaGridDependencySynchronize();
    bool absent = false;
    if (first + lane < a.rows) {
        const uint32_t key = uint32_t(first) + lane, at = first_not_below(a.sorted, a.places, key);
        absent = at == a.places || a.sorted[at].x != key;
    }
    O *out = reinterpret_cast<O *>(a.out);
    for (uint32_t m = __ballot_sync(0xffffffffu, absent); m; m &= m - 1) {
        O *row = out + (first + __ffs(int(m)) - 1) * a.width;
        for (uint64_t k = lane; k < a.width; k += 32) row[k] = to_element<O>(WideElement<OT>(0));
    }
}

// Sums through the norm of their rows: a cluster of 1 to 8 blocks for each row, 16 KB or more of it a block,
// which read both twice (the second time from L2); one division and one root a row, f64. `sums` may be the
// output itself. (Five rows of 512 KB among 138: a block each,
// by elements, 192 us a call; now 33.)
constexpr uint32_t kMostProject = 8;
struct Project {
    const char *table, *sums;
    char *out;
    const uint2 *sorted;
    uint64_t table_stride, width;
    uint32_t places, cleared; // rows without places are zero already
    uint32_t vectors;         // of a row
};

// N values of the wide type, as wide accesses as they allow.
template <class W, int N> __device__ __forceinline__ void load_values(W (&x)[N], const W *p) {
    constexpr int PART = sizeof(W) * N > 16 ? 16 / int(sizeof(W)) : N;
#pragma unroll
    for (int i = 0; i < N; i += PART) {
        Packed<W, PART> v;
        v.load(p + i);
#pragma unroll
        for (int e = 0; e < PART; ++e) x[i + e] = v.wide(e);
    }
}

template <uint32_t DT, int N>
__global__ void __launch_bounds__(kThreads) k_project(const __grid_constant__ Project a) {
    using T = Element<DT>;
    using W = WideElement<DT>;
    __shared__ double part[2][kWarps], total[2];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t size = cluster.num_blocks(), row = blockIdx.x / size;
    cudaGridDependencySynchronize();
    const uint32_t at = first_not_below(a.sorted, a.places, row);
    const uint32_t each = (a.vectors + size - 1) / size, lo = cluster.block_rank() * each, hi = min(a.vectors, lo + each);
    char *out = a.out + uint64_t(row) * a.width * sizeof(T);
    if (at == a.places || a.sorted[at].x != row) { // the same for the whole cluster
        if (a.cleared) return;
        Packed<T, N> none;
        none.fill(0);
        for (uint32_t k = lo + threadIdx.x; k < hi; k += kThreads) none.store(out + uint64_t(k) * Packed<T, N>::BYTES);
        return;
    }
    const char *table = a.table + uint64_t(row) * a.table_stride;
    const W *sums = reinterpret_cast<const W *>(a.sums) + uint64_t(row) * a.width;
    double tt = 0.0, tg = 0.0;
    const auto over_cluster = [&](auto &&join) { // of tt and tg
        for (int o = 16; o > 0; o >>= 1) {
            tt = join(tt, __shfl_xor_sync(0xffffffffu, tt, o));
            tg = join(tg, __shfl_xor_sync(0xffffffffu, tg, o));
        }
        if ((threadIdx.x & 31) == 0) {
            part[0][threadIdx.x >> 5] = tt;
            part[1][threadIdx.x >> 5] = tg;
        }
        __syncthreads();
        if (threadIdx.x < 2) {
            double all = 0.0;
            for (uint32_t w = 0; w < kWarps; ++w) all = join(all, part[threadIdx.x][w]);
            total[threadIdx.x] = all;
        }
        cluster.sync();
        tt = tg = 0.0;
        for (uint32_t b = 0; b < size; ++b) {
            const double *there = cluster.map_shared_rank(total, b);
            tt = join(tt, there[0]);
            tg = join(tg, there[1]);
        }
        cluster.sync(); // nobody leaves, or writes anew, while its sums are read
    };
    const auto add = [](double x, double y) { return x + y; };
#pragma unroll 4
    for (uint32_t k = lo + threadIdx.x; k < hi; k += kThreads) {
        Packed<T, N> t;
        W g[N];
        t.load(table + uint64_t(k) * Packed<T, N>::BYTES);
        load_values<W, N>(g, sums + uint64_t(k) * N);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const double x = t.wide(e);
            tt = fma(x, x, tt);
            tg = fma(x, double(g[e]), tg);
        }
    }
    over_cluster(add);
    if (out_of_range<W>(tt)) { // the same in the whole cluster
        const T *x = reinterpret_cast<const T *>(table);
        const uint32_t first = lo * N + threadIdx.x, end = hi * N;
        tt = 0.0;
#pragma unroll 1
        for (uint32_t k = first; k < end; k += kThreads) tt = fmax(tt, fabs(double(to_wide(x[k]))));
        over_cluster([](double v, double w) { return fmax(v, w); });
        const int power = power_of(tt);
        tt = tg = 0.0;
#pragma unroll 1
        for (uint32_t k = first; k < end; k += kThreads) {
            const double t = lowered(to_wide(x[k]), power);
            tt = fma(t, t, tt);
            tg = fma(t, double(sums[k]), tg);
        }
        over_cluster(add);
        const double inverse = tt == 0.0 ? 0.0 : 1.0 / sqrt(tt), along = tt == 0.0 ? 0.0 : tg / tt;
#pragma unroll 1
        for (uint32_t k = first; k < end; k += kThreads)
            reinterpret_cast<T *>(out)[k] = to_element<T>(
                W(lowered((double(sums[k]) - lowered(to_wide(x[k]), power) * along) * inverse, power)));
        return;
    }
    const double inverse = tt == 0.0 ? 0.0 : 1.0 / sqrt(tt), along = tt == 0.0 ? 0.0 : tg / tt;
#pragma unroll 4
    for (uint32_t k = lo + threadIdx.x; k < hi; k += kThreads) {
        Packed<T, N> t, y;
        W g[N];
        t.load(table + uint64_t(k) * Packed<T, N>::BYTES);
        load_values<W, N>(g, sums + uint64_t(k) * N);
#pragma unroll
        for (int e = 0; e < N; ++e) g[e] = W((double(g[e]) - double(t.wide(e)) * along) * inverse);
        y.pack(g);
        y.store(out + uint64_t(k) * Packed<T, N>::BYTES);
    }
}

// ------------------------------------------------------------------ few places: everything in one launch

// A block has `group` rows of the table. It lists the places that point to them, in order, and then a warp
// (a block for wide rows) sums each row's places, takes the sum through the norm, and writes the row,
// zeros where there is no place.
constexpr uint32_t kFewPlaces = 1024, kDirectVectors = 4;

struct Direct {
    const char *gradient, *table; // table: null unless rows are normalised
    char *out;
    Indices index;
    uint64_t stride, table_stride, row_bytes;
    double scale;
    uint32_t places, rows, group, vectors;
    uint32_t aligned; // vectors start on their size; otherwise they are moved by elements
};

template <class T, int N> __device__ __forceinline__ void load_any(Packed<T, N> &v, const char *p, uint32_t aligned) {
    if (aligned) return v.load(p);
    typename Packed<T, N>::W x[N];
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = to_wide(reinterpret_cast<const T *>(p)[e]);
    v.pack(x);
}

template <uint32_t DT, int N, bool BLOCK>
__global__ void __launch_bounds__(kThreads, 2) k_direct(const __grid_constant__ Direct a) {
    using T = Element<DT>;
    using W = WideElement<DT>;
    __shared__ uint32_t list[kFewPlaces]; // the row within the group << 16 | the place
    __shared__ uint32_t count[kWarps + 1];
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const uint32_t row0 = blockIdx.y * a.group, rows = min(a.group, a.rows - row0);
    const uint32_t each = (a.places + kThreads - 1) / kThreads * 32, lo = warp * each; // places of a warp
    constexpr uint32_t ROUNDS = kFewPlaces / kThreads;
    uint32_t mine[ROUNDS], found = 0;
#pragma unroll
    for (uint32_t j = 0; j < ROUNDS; ++j) {
        const uint32_t i = lo + j * 32 + lane;
        mine[j] = j * 32 < each && i < a.places ? key_at(a.index, i) - row0 : kAbsent;
        found += __popc(__ballot_sync(0xffffffffu, mine[j] < rows));
    }
    if (lane == 0) count[warp] = found;
    __syncthreads();
    uint32_t at = 0, all = 0;
    for (uint32_t w = 0; w < kWarps; ++w) {
        if (w == warp) at = all;
        all += count[w];
    }
#pragma unroll
    for (uint32_t j = 0; j < ROUNDS; ++j) {
        const uint32_t here = __ballot_sync(0xffffffffu, mine[j] < rows);
        if (mine[j] < rows) list[at + __popc(here & ((1u << lane) - 1))] = mine[j] << 16 | (lo + j * 32 + lane);
        at += __popc(here);
    }
    __syncthreads();
    // places at a time: four in registers left one block on an SM (22 us instead of 17 for 1024 places of 509
    // rows of 16 KB)
    constexpr uint32_t THREADS = BLOCK ? kThreads : 32, PLACES = Packed<T, N>::BYTES == 16 ? 2 : 4;
    const uint32_t thread = BLOCK ? t : lane, vector0 = blockIdx.x * (THREADS * kDirectVectors) + thread;
    for (uint32_t r = BLOCK ? 0 : warp; r < rows; r += BLOCK ? 1 : kWarps) {
        W sum[kDirectVectors][N];
#pragma unroll
        for (uint32_t j = 0; j < kDirectVectors; ++j)
#pragma unroll
            for (int e = 0; e < N; ++e) sum[j][e] = W(0);
        bool any = false;
        for (uint32_t b = 0; b < all; b += 32) {
            const uint32_t entry = b + lane < all ? list[b + lane] : kAbsent;
            uint32_t same = __ballot_sync(0xffffffffu, b + lane < all && entry >> 16 == r);
            any = any || same;
            while (same) {
                Packed<T, N> v[PLACES][kDirectVectors];
                uint32_t n = 0;
#pragma unroll
                for (uint32_t q = 0; q < PLACES; ++q) {
                    if (!same) break;
                    const uint32_t place = __shfl_sync(0xffffffffu, entry, __ffs(int(same)) - 1) & 0xffff;
                    same &= same - 1;
                    ++n;
                    const char *from = a.gradient + uint64_t(place) * a.stride;
#pragma unroll
                    for (uint32_t j = 0; j < kDirectVectors; ++j) {
                        const uint32_t k = vector0 + j * THREADS;
                        if (k < a.vectors) load_any<T, N>(v[q][j], from + uint64_t(k) * Packed<T, N>::BYTES, a.aligned);
                    }
                }
#pragma unroll
                for (uint32_t q = 0; q < PLACES; ++q)
                    if (q < n)
#pragma unroll
                        for (uint32_t j = 0; j < kDirectVectors; ++j)
                            if (vector0 + j * THREADS < a.vectors)
#pragma unroll
                                for (int e = 0; e < N; ++e) sum[j][e] += v[q][j].wide(e);
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < kDirectVectors; ++j)
#pragma unroll
            for (int e = 0; e < N; ++e) sum[j][e] *= W(a.scale);
        const uint64_t row = uint64_t(row0) + r;
        double along = 0.0, inverse = 1.0;
        Packed<T, N> unit[kDirectVectors];
        if (a.table && any) { // the same in all threads of the row
            const char *from = a.table + row * a.table_stride;
            double tt = 0.0, ts = 0.0;
#pragma unroll
            for (uint32_t j = 0; j < kDirectVectors; ++j) {
                const uint32_t k = vector0 + j * THREADS;
                if (k >= a.vectors) continue;
                load_any<T, N>(unit[j], from + uint64_t(k) * Packed<T, N>::BYTES, a.aligned);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const double x = unit[j].wide(e);
                    tt = fma(x, x, tt);
                    ts = fma(x, double(sum[j][e]), ts);
                }
            }
            tt = sum_over<BLOCK>(tt, 32);
            if constexpr (BLOCK) __syncthreads(); // the first sum's shared memory
            ts = sum_over<BLOCK>(ts, 32);
            if constexpr (BLOCK) __syncthreads();
            if (out_of_range<W>(tt)) {
                double largest = 0.0;
#pragma unroll
                for (uint32_t j = 0; j < kDirectVectors; ++j)
                    if (vector0 + j * THREADS < a.vectors)
#pragma unroll
                        for (int e = 0; e < N; ++e) largest = fmax(largest, fabs(double(unit[j].wide(e))));
                const int power = power_of(largest_over<BLOCK>(largest, 32));
                tt = ts = 0.0;
#pragma unroll
                for (uint32_t j = 0; j < kDirectVectors; ++j) {
                    if (vector0 + j * THREADS >= a.vectors) continue;
                    rescale(unit[j], power);
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const double x = unit[j].wide(e);
                        sum[j][e] = W(lowered(sum[j][e], power)); // what is over the norm goes on so
                        tt = fma(x, x, tt);
                        ts = fma(x, double(sum[j][e]), ts);
                    }
                }
                tt = sum_over<BLOCK>(tt, 32);
                if constexpr (BLOCK) __syncthreads();
                ts = sum_over<BLOCK>(ts, 32);
                if constexpr (BLOCK) __syncthreads();
            }
            inverse = tt == 0.0 ? 0.0 : 1.0 / sqrt(tt);
            along = tt == 0.0 ? 0.0 : ts / tt;
        }
#pragma unroll
        for (uint32_t j = 0; j < kDirectVectors; ++j) {
            const uint32_t k = vector0 + j * THREADS;
            if (k >= a.vectors) continue;
            Packed<T, N> y;
            W x[N];
#pragma unroll
            for (int e = 0; e < N; ++e)
                x[e] = a.table && any ? W((double(sum[j][e]) - double(unit[j].wide(e)) * along) * inverse) : sum[j][e];
            y.pack(x);
            char *to = a.out + row * a.row_bytes + uint64_t(k) * Packed<T, N>::BYTES;
            if (a.aligned) y.store(to);
            else
#pragma unroll
                for (int e = 0; e < N; ++e) reinterpret_cast<T *>(to)[e] = to_element<T>(y.wide(e));
        }
    }
}

// ------------------------------------------------------------------ host

[[noreturn]] void refuse(const char *what, const char *why) {
    fail(std::string("the embedding's ") + what + " " + why);
}

void check_rows(const ArcqmlRows &r, const char *what) {
    if (r.dtype > ARCQML_F16) refuse(what, "has an unknown type");
    if (r.reserved != 0) refuse(what, "has a nonzero reserved field");
    if (r.rows >> 31) refuse(what, "has too many rows (below 2^31)");
    if (r.width == 0) refuse(what, "has rows without elements");
    if (r.width >> 30) refuse(what, "has rows that are too long (below 2^30 elements)");
    if (r.stride >> 40) refuse(what, "has rows too far apart");
    // (accesses are as wide as all addresses allow, so that of no rows has to start on an element too)
    if (reinterpret_cast<uintptr_t>(r.data) % bytes_of_element(r.dtype))
        refuse(what, "is not aligned to its elements");
    if (r.rows && !r.data) refuse(what, "is null");
}

void check_options(const ArcqmlEmbeddingOptions &o) {
    if (!std::isfinite(o.scale)) refuse("scale", "must be finite");
    if (o.normalize != 0 && o.normalize != 1) refuse("options", "are invalid (normalize is 0 or 1)");
    if (o.index_bytes != 4 && o.index_bytes != 8) refuse("indices", "must have 4 or 8 bytes");
}

void check_indices(const void *indices, size_t count, const ArcqmlEmbeddingOptions &o) {
    if (count >> 31) refuse("indices", "are too many (below 2^31)");
    if (!count) return;
    if (!indices) refuse("indices", "are null");
    if (reinterpret_cast<uintptr_t>(indices) % size_t(o.index_bytes)) refuse("indices", "are not aligned");
}

void check_scratch(const double *ws, size_t len, size_t need) {
    if (!need) return;
    if (!ws) fail("workspace is null");
    if (reinterpret_cast<uintptr_t>(ws) % 16) fail("workspace is not aligned to 16 bytes");
    if (len < need) {
        std::ostringstream m;
        m << "workspace of " << len << " doubles is too small: the call needs " << need;
        fail(m.str());
    }
}

uint32_t power_of_two_from(uint64_t n) {
    uint32_t p = 1;
    while (p < n && p < 32) p *= 2;
    return p;
}

// The largest access, up to 16 bytes, on which every row starts and ends.
uint32_t access_bytes(uint64_t bits) {
    uint32_t v = 16;
    while (v > 1 && bits % v) v /= 2;
    return v;
}

// f(type code, elements of an access), for what an access of `bytes` can hold.
template <class F> void for_access(uint32_t dtype, uint32_t bytes, F &&f) {
    const auto pick = [&](auto type) {
        constexpr uint32_t DT = type, SIZE = sizeof(Element<DT>);
        if constexpr (SIZE <= 2)
            if (bytes == 2) return f(type, std::integral_constant<int, 2 / SIZE>{});
        if constexpr (SIZE <= 4)
            if (bytes == 4) return f(type, std::integral_constant<int, 4 / SIZE>{});
        if (bytes == 8) return f(type, std::integral_constant<int, 8 / SIZE>{});
        return f(type, std::integral_constant<int, 16 / SIZE>{});
    };
    switch (dtype) {
    case ARCQML_F64: return pick(std::integral_constant<uint32_t, ARCQML_F64>{});
    case ARCQML_F32: return pick(std::integral_constant<uint32_t, ARCQML_F32>{});
    case ARCQML_BF16: return pick(std::integral_constant<uint32_t, ARCQML_BF16>{});
    default: return pick(std::integral_constant<uint32_t, ARCQML_F16>{});
    }
}

struct Shape {
    uint64_t blocks;
    uint32_t threads;
    bool follows = false; // may start while the call's last launch ends
    uint32_t cluster = 1, shared = 0, down = 1; // down: the grid's second dimension
};

template <class... P, class... A>
void start(void (*kernel)(P...), const Shape &shape, double bytes, cudaStream_t s, const A &...args) {
    if (shape.blocks >> 31 || shape.down > 65535) fail("the embedding call is too large for one launch");
    cudaLaunchConfig_t c{};
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = shape.cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    c.attrs = shape.follows ? at : at + 1;
    c.numAttrs = (shape.follows ? 1 : 0) + (shape.cluster > 1 ? 1 : 0);
    c.gridDim = dim3(uint32_t(shape.blocks), shape.down);
    c.blockDim = dim3(shape.threads);
    c.dynamicSmemBytes = shape.shared;
    c.stream = s;
    std::tuple<P...> held{P(args)...};
    const ProfToken tok = prof_begin(PROF_OTHER, s);
    const cudaError_t e = std::apply([&](auto &...x) { return cudaLaunchKernelEx(&c, kernel, x...); }, held);
    check_cuda(e, "embedding kernel launch");
    prof_end(tok, s, bytes);
}

// Lets the sort have clusters of 16 blocks, once on each device.
template <auto KERNEL> void allow_cluster() {
    static std::atomic<uint64_t> set{0};
    int device = 0;
    check_cuda(cudaGetDevice(&device), "cudaGetDevice");
    if (device < 64 && (set.load() >> device & 1)) return;
    check_cuda(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "embedding kernel attribute");
    if (device < 64) set |= uint64_t(1) << device;
}

uint64_t blocks_for(uint64_t threads) { return (threads + kThreads - 1) / kThreads; }

uint64_t address(const void *p) { return reinterpret_cast<uintptr_t>(p); }

// The most pieces that a normalised row may be cut into (0: its threads hold it): accesses are as small as
// an element where rows start anywhere.
uint32_t most_pieces(const ArcqmlRows &t, const ArcqmlEmbeddingOptions &o) {
    return o.normalize && t.width > kThreads * kRowVectors ? uint32_t((t.width + kPieceVectors - 1) / kPieceVectors) : 0;
}

// Scratch of the gradient, in 4-byte words from its start.
struct GradientScratch {
    uint64_t sorted[2], counts, totals, partial, sums, words;
    uint32_t blocks, passes, bits, chunk, chunks;
};

GradientScratch gradient_scratch(const ArcqmlRows &g, uint64_t rows, const ArcqmlEmbeddingOptions &o) {
    GradientScratch s{};
    const uint64_t n = g.rows;
    // few places, and not many to a row: one launch. A row that goes through its norm has to fit into a block.
    const uint64_t row = g.width * bytes_of_element(g.dtype);
    if (n <= kFewPlaces && n <= 16 * rows && (!o.normalize || row / access_bytes(row | 16) <= kThreads * kDirectVectors))
        return s;
    const auto take = [&](uint64_t words) {
        const uint64_t at = s.words;
        s.words += (words + 3) / 4 * 4;
        return at;
    };
    uint32_t bits = 1;
    while (bits < 32 && (rows >> bits)) ++bits; // kAbsent's digits are all ones: above any row's
    s.passes = (bits + 8) / 9;
    s.bits = (bits + s.passes - 1) / s.passes;
    s.blocks = uint32_t((n + kSortKeys - 1) / kSortKeys);
    const bool in_cluster = n <= kMostPerThread * kClusterThreads * kMostCluster;
    for (int i = 0; i < 2; ++i) {
        s.sorted[i] = take(2 * n);
    }
    if (!in_cluster) {
        s.counts = take(uint64_t(s.passes) * s.blocks * kBins);
        s.totals = take(kBins);
    }
    // chunks of 8 to 128 places: enough of them to fill the GPU, and not more than 2048 beyond that, since a row
    // that many places point to is put together from its chunks (131071 places of 128 bytes took 46 us for
    // that in chunks of 8, 27 us in chunks of 32)
    const uint64_t tiles = std::max<uint64_t>(1, g.width * bytes_of_element(g.dtype) / 512);
    s.chunk = 8;
    while (s.chunk < 128 && (n * tiles / (s.chunk * 2) >= 148 * 32 || n / s.chunk > 2048)) s.chunk *= 2;
    s.chunks = uint32_t((n + s.chunk - 1) / s.chunk);
    const uint64_t wide = g.dtype == ARCQML_F64 ? 2 : 1;
    s.partial = take(2 * uint64_t(s.chunks) * g.width * wide);
    s.sums = s.words;
    if (o.normalize && (g.dtype == ARCQML_BF16 || g.dtype == ARCQML_F16)) take(rows * g.width);
    return s;
}

}  // namespace

size_t embedding_lookup_workspace(const ArcqmlRows &table, size_t count, const ArcqmlEmbeddingOptions &o) {
    return size_t(most_pieces(table, o)) * count * (table.dtype == ARCQML_F64 ? 2 : 1);
}

size_t embedding_gradient_workspace(const ArcqmlRows &gradient, uint64_t rows, const ArcqmlEmbeddingOptions &o) {
    return size_t((gradient_scratch(gradient, rows, o).words + 1) / 2);
}

void embedding_lookup_device(const ArcqmlRows &table, const void *indices, size_t count,
                             const ArcqmlEmbeddingOptions &o, const ArcqmlRows &out, double *ws,
                             size_t ws_len, cudaStream_t s) {
    check_options(o);
    check_rows(table, "table");
    check_rows(out, "output");
    check_indices(indices, count, o);
    if (out.dtype != table.dtype || out.width != table.width || out.rows != count || out.stride != out.width)
        refuse("output", "does not have the table's type and width, a row for each index and no gaps");
    check_scratch(ws, ws_len, embedding_lookup_workspace(table, count, o));
    if (!count) return;
    const uint64_t size = bytes_of_element(table.dtype);
    Lookup a{};
    a.table = static_cast<const char *>(table.data);
    a.out = static_cast<char *>(out.data);
    a.index = {indices, table.rows, o.padding, o.index_bytes == 8};
    a.places = count;
    a.stride = table.stride * size;
    a.row_bytes = table.width * size;
    a.scale = o.scale;
    const uint32_t bytes = access_bytes(address(table.data) | address(out.data) | a.stride | a.row_bytes | 16);
    const uint64_t vectors = a.row_bytes / bytes;
    a.vectors = uint32_t(vectors);
    const double moved = 2.0 * double(count) * double(a.row_bytes);
    const bool held = o.normalize && vectors <= kThreads * kRowVectors;
    for_access(table.dtype, bytes, [&](auto type, auto n) {
        constexpr uint32_t DT = type;
        constexpr int N = n;
        if (held && vectors > 32 * kRowVectors) return start(k_lookup_row<DT, N, true>, {count, kThreads}, moved, s, a);
        if (held) {
            a.lanes = power_of_two_from((vectors + 1) / 2);
            while (a.lanes * kRowVectors < vectors) a.lanes *= 2;
            return start(k_lookup_row<DT, N, false>, {blocks_for(count * a.lanes), kThreads}, moved, s, a);
        }
        if (o.normalize) {
            a.pieces = uint32_t((vectors + kPieceVectors - 1) / kPieceVectors);
            start(k_row_squares<DT, N>, {count * a.pieces, kThreads}, moved / 2, s, a, ws);
            a.squares = ws;
        }
        a.lanes = power_of_two_from((vectors + kTileVectors - 1) / kTileVectors);
        a.tiles = uint32_t((vectors + a.lanes * kTileVectors - 1) / (a.lanes * kTileVectors));
        start(k_lookup<DT, N>, {blocks_for(count * a.tiles * a.lanes), kThreads}, moved, s, a);
    });
}

void embedding_gradient_device(const ArcqmlRows &gradient, const void *indices, const ArcqmlEmbeddingOptions &o,
                               const ArcqmlRows *table, const ArcqmlRows &out, double *ws, size_t ws_len,
                               cudaStream_t s) {
    check_options(o);
    check_rows(gradient, "gradient");
    check_rows(out, "output");
    check_indices(indices, gradient.rows, o);
    if (out.dtype != gradient.dtype || out.width != gradient.width || out.stride != out.width)
        refuse("output", "does not have the gradient's type and width, without gaps");
    if (o.normalize && !table) refuse("table", "is null and its rows are normalised");
    if (!o.normalize && table) refuse("table", "is given and its rows are not normalised");
    if (table) {
        check_rows(*table, "table");
        if (table->dtype != out.dtype || table->width != out.width || table->rows != out.rows)
            refuse("table", "does not have the output's type and shape");
    }
    const uint64_t size = bytes_of_element(gradient.dtype), n = gradient.rows, row = out.width * size;
    const GradientScratch w = gradient_scratch(gradient, out.rows, o);
    check_scratch(ws, ws_len, size_t((w.words + 1) / 2));
    if (!out.rows) return;
    const uint64_t starts = address(gradient.data) | address(out.data) | gradient.stride * size | row | 16;
    const uint32_t bytes = access_bytes(table ? starts | address(table->data) | table->stride * size : starts);
    const Indices index{indices, out.rows, o.padding, o.index_bytes == 8};
    const double moved = double(n) * double(row);
    if (!w.words) {
        Direct a{};
        a.gradient = static_cast<const char *>(gradient.data);
        a.table = table ? static_cast<const char *>(table->data) : nullptr;
        a.out = static_cast<char *>(out.data);
        a.index = index;
        a.stride = gradient.stride * size;
        a.table_stride = table ? table->stride * size : 0;
        a.row_bytes = row;
        a.scale = o.scale;
        a.places = uint32_t(n);
        a.rows = uint32_t(out.rows);
        const uint32_t whole = access_bytes(row | 16);
        a.aligned = bytes == whole;
        a.vectors = uint32_t(row / whole);
        const bool wide = a.vectors > 32 * kDirectVectors;
        const uint32_t across = wide ? (a.vectors + kThreads * kDirectVectors - 1) / (kThreads * kDirectVectors) : 1;
        // blocks for each place on the GPU; warps take the rows of a block in turn. At most 32769 blocks of rows,
        // in the grid's second dimension; the pieces of a row, up to 2^20, have the first one
        a.group = uint32_t(std::min<uint64_t>(65535, (out.rows + 148 * 6 - 1) / (148 * 6)));
        if (!wide) a.group = std::max(a.group, kWarps);
        const Shape shape{across, kThreads, false, 1, 0, uint32_t((out.rows + a.group - 1) / a.group)};
        return for_access(gradient.dtype, whole, [&](auto type, auto nn) {
            constexpr uint32_t DT = type;
            constexpr int N = nn;
            if (wide) start(k_direct<DT, N, true>, shape, moved, s, a);
            else start(k_direct<DT, N, false>, shape, moved, s, a);
        });
    }
    uint32_t *base = reinterpret_cast<uint32_t *>(ws);
    const bool in_cluster = n <= kMostPerThread * kClusterThreads * kMostCluster;
    uint2 *buffers[2] = {reinterpret_cast<uint2 *>(base + w.sorted[0]), reinterpret_cast<uint2 *>(base + w.sorted[1])};
    const uint2 *sorted = buffers[in_cluster ? 0 : w.passes & 1];
    if (in_cluster) {
        ClusterSort a{};
        a.index = index;
        a.out[0] = buffers[0];
        a.out[1] = buffers[1];
        a.clear = static_cast<char *>(out.data);
        a.clear_bytes = out.rows * row;
        a.places = uint32_t(n);
        a.passes = w.passes;
        a.bits = w.bits;
        const auto sort = [&](auto per_thread) {
            constexpr uint32_t P = per_thread;
            uint32_t cluster = 1;
            while (cluster * P * kClusterThreads < n) cluster *= 2;
            allow_cluster<k_sort_cluster<P>>();
            // as many blocks clear as the GPU takes beside the sort, at least 64 KB each
            const uint64_t clears = std::min<uint64_t>((112 - cluster) / cluster, a.clear_bytes / (uint64_t(cluster) << 16) + 1);
            start(k_sort_cluster<P>, {cluster * (1 + clears), kClusterThreads, false, cluster, sizeof(ClusterShared)},
                  double(a.clear_bytes), s, a);
        };
        const uint32_t each = kClusterThreads * kMostCluster;
        if (n <= each) sort(std::integral_constant<uint32_t, 1>{});
        else if (n <= 2 * each) sort(std::integral_constant<uint32_t, 2>{});
        else if (n <= 4 * each) sort(std::integral_constant<uint32_t, 4>{});
        else sort(std::integral_constant<uint32_t, 8>{});
    } else {
        Sort a{};
        a.index = index;
        a.places = uint32_t(n);
        a.blocks = w.blocks;
        a.bits = w.bits;
        const uint64_t each = uint64_t(w.blocks) * kBins;
        a.counts = base + w.counts;
        a.next = a.counts + each;
        start(k_count_digits, {w.blocks, kThreads}, 8.0 * double(n), s, a, each * (w.passes - 1));
        for (uint32_t p = 0; p < w.passes; ++p) {
            a.shift = p * w.bits;
            a.next_shift = a.shift + w.bits;
            a.counts = base + w.counts + p * each;
            a.next = p + 1 < w.passes ? a.counts + each : nullptr;
            a.from = p ? buffers[p & 1] : nullptr;
            a.out = buffers[(p + 1) & 1];
            a.totals = nullptr;
            if (w.blocks > 128) {
                a.totals = base + w.totals;
                start(k_prefix_counts, {kBins / 32, 1024, true}, 8.0 * double(each), s, a.counts, a.totals, w.blocks);
            }
            start(k_sort_pass, {w.blocks, kThreads, true}, 16.0 * double(n), s, a);
        }
    }
    Sums a{};
    a.gradient = static_cast<const char *>(gradient.data);
    a.sorted = sorted;
    a.partial = base + w.partial;
    a.stride = gradient.stride * size;
    a.width = out.width;
    a.rows = out.rows;
    a.scale = o.scale;
    a.places = uint32_t(n);
    a.chunk = w.chunk;
    a.chunks = w.chunks;
    const bool apart = o.normalize && size == 2; // the sums keep 32 bits until the norm is through
    a.out = apart ? reinterpret_cast<char *>(base + w.sums) : static_cast<char *>(out.data);
    a.vectors = uint32_t(row / bytes);
    a.lanes = power_of_two_from(a.vectors);
    a.tiles = (a.vectors + a.lanes - 1) / a.lanes;
    for_access(gradient.dtype, bytes, [&](auto type, auto nn) {
        constexpr uint32_t DT = type;
        constexpr int N = nn;
        constexpr uint32_t WIDE = DT == ARCQML_F64 ? ARCQML_F64 : ARCQML_F32;
        const auto sums = [&](auto kind) {
            constexpr uint32_t OT = kind;
            if (!n) return;
            const Shape shape{blocks_for(uint64_t(a.chunks) * a.tiles * a.lanes), kThreads, true};
            start(k_sum_chunks<DT, OT, N>, shape, moved, s, a);
            if (a.chunks > 1)
                start(k_join_chunks<DT, OT, N>, {uint64_t(a.chunks - 1) * ((a.vectors + 31) / 32), kThreads, true}, 0.0, s, a);
        };
        if constexpr (WIDE != DT) {
            if (apart) sums(std::integral_constant<uint32_t, WIDE>{});
            else sums(type);
        } else {
            sums(type);
        }
    });
    if (!o.normalize) {
        if (!in_cluster)
            for_access(out.dtype, 16, [&](auto type, auto) {
                constexpr uint32_t DT = type;
                start(k_zero_rows<DT>, {(out.rows + kWarps * 32 - 1) / (kWarps * 32), kThreads, true}, 0.0, s, a);
            });
        return;
    }
    Project p{};
    p.table = static_cast<const char *>(table->data);
    p.sums = a.out;
    p.out = static_cast<char *>(out.data);
    p.sorted = sorted;
    p.table_stride = table->stride * size;
    p.width = out.width;
    p.places = uint32_t(n);
    p.cleared = in_cluster;
    p.vectors = uint32_t(row / bytes);
    uint32_t cluster = 1;
    while (cluster < kMostProject && row >= uint64_t(cluster) << 15) cluster *= 2;
    for_access(out.dtype, bytes, [&](auto type, auto nn) {
        constexpr uint32_t DT = type;
        constexpr int N = nn;
        start(k_project<DT, N>, {out.rows * cluster, kThreads, true, cluster}, 3.0 * double(row) * double(out.rows), s, p);
    });
}

}  // namespace arcqml
