// Rows ordered by a small integer key (expert or table id): a stable least-significant-digit radix sort of
// (key, index) pairs, and the key offsets.  Every place follows from counts alone, so the order is the same in
// every run.
#include "rows.cuh"
#include "odie_b200.h"

namespace odie {
namespace {

// A tile of pairs per block of 256 threads.  Warp w holds the tile's pairs [w * 32 R, (w + 1) * 32 R) in R
// rounds of 32, lane order within a round, so that (warp, round, lane) is the input order.
constexpr int THREADS = 256, WARPS = THREADS / 32;
// Up to 128 tiles, every block sums the counts of the tiles before its own itself (32 tiles: 6.5 us with that, 8.8 in
// two kernels; 512 tiles take the kernel between).
constexpr int ROUNDS = 8, TILE = THREADS * ROUNDS, FOLD = 128;
// One block orders up to 4096 pairs by itself; more are cut into tiles of 2048.  (A block of 1024 threads for up to 16384
// saved a launch and took 19 us where two kernels take 9.)
constexpr int ONE_ROUNDS = 16, ONE_TILE = THREADS * ONE_ROUNDS;
// Digits of up to 10 bits: two passes order 2^20 keys, one pass 1023 experts, and the eight warps' counts fit
// in 32 KB of shared memory.
constexpr int MAX_DIGIT_BITS = 10;

int key_bits(int bins) {  // keys 0..bins
    int bits = 1;
    while ((int64_t(1) << bits) <= bins) ++bits;
    return bits;
}
int pass_count(int bins) { return (key_bits(bins) + MAX_DIGIT_BITS - 1) / MAX_DIGIT_BITS; }
int digit_bits(int bins) { return (key_bits(bins) + pass_count(bins) - 1) / pass_count(bins); }

// SOURCE: where a pass finds its pairs: 4 or 8, the caller's int32 or int64 keys, or 0, the pairs of the pass before.
template <int SOURCE>
__device__ __forceinline__ uint32_t read_key(const void* keys, long long i, uint32_t bins) {
    if (SOURCE == 8) {
        const long long k = __ldg(static_cast<const long long*>(keys) + i);
        return k >= 0 && k < (long long)bins ? uint32_t(k) : bins;
    }
    if (SOURCE == 4) {
        const int k = __ldg(static_cast<const int*>(keys) + i);
        return k >= 0 && k < int(bins) ? uint32_t(k) : bins;
    }
    return __ldg(static_cast<const uint32_t*>(keys) + i);
}

// Exclusive sum over the block's threads; total gets the sum of all.  scratch: WARPS words of shared memory.
__device__ __forceinline__ uint32_t block_exclusive(uint32_t v, uint32_t* scratch, uint32_t& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t sum = v;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const uint32_t other = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += other;
    }
    if (lane == 31) scratch[warp] = sum;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += scratch[w];
        total += scratch[w];
    }
    __syncthreads();
    return before + sum - v;
}

// The lanes of the warp whose digit of `bits` bits is this lane's, among those that are on: a ballot per bit
// (7 us less than match.any for 64 experts: that instruction takes one turn per distinct value).
__device__ __forceinline__ uint32_t digit_peers(uint32_t d, bool on, int bits) {
    uint32_t peers = __ballot_sync(0xffffffffu, on);
    for (int b = 0; b < bits; ++b) {
        const bool bit = (d >> b) & 1;
        const uint32_t ones = __ballot_sync(0xffffffffu, bit);
        peers &= bit ? ones : ~ones;
    }
    return peers;
}

// Ranks of the tile's pairs among those with the same digit in their own warp, in input order; the warps' digit
// counts are left in counts[warp][digits].
template <int R>
__device__ __forceinline__ void warp_ranks(const uint32_t (&key)[R], int rounds, int live, int shift, int bits, uint32_t* counts,
                                           uint32_t (&rank)[R]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, digits = 1 << bits;
    for (int i = threadIdx.x; i < WARPS * digits; i += THREADS) counts[i] = 0;
    __syncthreads();
    uint32_t* mine = counts + warp * digits;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r >= rounds) break;
        const bool on = (warp * rounds + r) * 32 + lane < live;
        const uint32_t d = (key[r] >> shift) & uint32_t(digits - 1);
        const uint32_t peers = digit_peers(d, on, bits);
        const uint32_t before = on ? mine[d] : 0;
        __syncwarp();
        rank[r] = before + __popc(peers & ((1u << lane) - 1));
        if (on && (peers >> lane) == 1u) mine[d] = before + __popc(peers);  // the last lane of the peers
        __syncwarp();
    }
    __syncthreads();
}

// counts[warp][digit] becomes first[digit] + the pairs of that digit in earlier warps.
__device__ __forceinline__ void warp_starts(uint32_t* counts, int digits, const uint32_t* first) {
    for (int d = threadIdx.x; d < digits; d += THREADS) {
        uint32_t at = first[d];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const uint32_t c = counts[w * digits + d];
            counts[w * digits + d] = at;
            at += c;
        }
    }
    __syncthreads();
}

// All of it in one block, for at most one tile: a step's few rows cost one launch.
template <int SOURCE>
__global__ void __launch_bounds__(THREADS) sort_tile_kernel(SortArgs a, int passes, int bits) {
    extern __shared__ uint32_t shared[];
    const int digits = 1 << bits, n = int(a.n);
    uint32_t* counts = shared;                    // [WARPS][digits]
    uint32_t* first = counts + WARPS * digits;    // [digits]
    uint32_t* index = first + digits;             // [ONE_TILE]
    uint32_t* keys = index + ONE_TILE;            // [ONE_TILE], of several passes or where they are wanted
    const bool keep_keys = passes > 1 || a.sorted;
    __shared__ uint32_t scan[WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rounds = (n + THREADS - 1) / THREADS;
    uint32_t key[ONE_ROUNDS], id[ONE_ROUNDS], rank[ONE_ROUNDS];
#pragma unroll
    for (int r = 0; r < ONE_ROUNDS; ++r) {
        const int i = (warp * rounds + r) * 32 + lane;
        key[r] = r < rounds ? read_key<SOURCE>(a.keys, min(i, n - 1), uint32_t(a.bins)) : 0;
        id[r] = uint32_t(i);
    }
    for (int p = 0; p < passes; ++p) {
        warp_ranks(key, rounds, n, p * bits, bits, counts, rank);
        uint32_t running = 0;
        for (int base = 0; base < digits; base += THREADS) {
            const int d = base + threadIdx.x;
            uint32_t c = 0, total;
            if (d < digits)
                for (int w = 0; w < WARPS; ++w) c += counts[w * digits + d];
            const uint32_t before = block_exclusive(c, scan, total);
            if (d < digits) first[d] = running + before;
            running += total;
        }
        __syncthreads();
        if (passes == 1 && a.offsets)
            for (int d = threadIdx.x; d <= a.bins; d += THREADS) a.offsets[d] = int(first[d]);
        warp_starts(counts, digits, first);
        const bool last = p + 1 == passes;
#pragma unroll
        for (int r = 0; r < ONE_ROUNDS; ++r) {
            const int i = (warp * rounds + r) * 32 + lane;
            if (r < rounds && i < n) {
                const uint32_t place = counts[warp * digits + ((key[r] >> (p * bits)) & uint32_t(digits - 1))] + rank[r];
                const bool kept = key[r] < uint32_t(a.bins);
                index[place] = last && !kept ? ~id[r] : id[r];
                if (keep_keys) keys[place] = key[r];
                if (last && a.slot) a.slot[id[r]] = kept ? int(place) : ~int(place);
            }
        }
        __syncthreads();
        if (last) break;
#pragma unroll
        for (int r = 0; r < ONE_ROUNDS; ++r) {
            const int i = (warp * rounds + r) * 32 + lane;
            if (r < rounds && i < n) {
                key[r] = keys[i];
                id[r] = index[i];
            }
        }
        __syncthreads();
    }
    // out through shared memory, in order
    for (int i = threadIdx.x; i < n; i += THREADS) {
        a.order[i] = int(index[i]);
        if (a.sorted) a.sorted[i] = keys[i];
    }
    if (passes > 1 && a.offsets) {
        for (int d = threadIdx.x; d <= a.bins; d += THREADS) {
            int lo = 0, hi = n;
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (keys[mid] < uint32_t(d)) lo = mid + 1;
                else hi = mid;
            }
            a.offsets[d] = lo;
        }
    }
}

struct Pass {
    const void* keys;           // first pass: the caller's, later the pairs of the pass before
    const uint32_t* index;
    uint32_t* keys_out;         // null in the last pass
    uint32_t* index_out;
    uint32_t* tiles;            // [tile][digit]: counts, then the pairs of that digit in earlier tiles
    uint32_t* totals;           // [digit]
    int shift, bits;
};

template <int SOURCE>
__global__ void __launch_bounds__(THREADS) tile_counts_kernel(SortArgs a, Pass p) {
    extern __shared__ uint32_t shared[];
    const int digits = 1 << p.bits;
    for (int d = threadIdx.x; d < digits; d += THREADS) shared[d] = 0;
    __syncthreads();
    const long long begin = (long long)blockIdx.x * TILE;
    uint32_t key[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        key[r] = read_key<SOURCE>(p.keys, min(begin + (long long)(r * THREADS + threadIdx.x), (long long)a.n - 1), uint32_t(a.bins));
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {  // lanes with one digit add once
        const bool on = begin + r * THREADS + threadIdx.x < a.n;
        const uint32_t d = (key[r] >> p.shift) & uint32_t(digits - 1), peers = digit_peers(d, on, p.bits);
        if (on && (peers >> (threadIdx.x & 31)) == 1u) atomicAdd(shared + d, __popc(peers));
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += THREADS) p.tiles[(long long)blockIdx.x * digits + d] = shared[d];
}

// A block per 32 digits: lane = digit, warp w sums its share of the tiles, then writes their starts.
__global__ void __launch_bounds__(1024) tile_starts_kernel(Pass p, int tiles) {
    __shared__ uint32_t sums[32][33];
    const int digits = 1 << p.bits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int d = blockIdx.x * 32 + lane, share = (tiles + 31) / 32;
    const int from = min(tiles, warp * share), to = min(tiles, from + share);
    uint32_t sum = 0;
    if (d < digits) {
#pragma unroll 8
        for (int t = from; t < to; ++t) sum += p.tiles[(long long)t * digits + d];
    }
    sums[warp][lane] = sum;
    __syncthreads();
    uint32_t at = 0, total = 0;
    for (int w = 0; w < 32; ++w) {
        if (w < warp) at += sums[w][lane];
        total += sums[w][lane];
    }
    if (d < digits) {
        if (warp == 0) p.totals[d] = total;
#pragma unroll 8
        for (int t = from; t < to; ++t) {
            const uint32_t c = p.tiles[(long long)t * digits + d];
            p.tiles[(long long)t * digits + d] = at;
            at += c;
        }
    }
}

// tiles: their count where the blocks sum the counts of earlier tiles, 0 where tile_starts_kernel did.
// The tile's pairs are put in digit order in shared memory first, so that neighbouring threads write neighbouring
// places (2^20 pairs of 16384 ids: 15 us a pass written straight to their places).
template <int SOURCE>
__global__ void __launch_bounds__(THREADS) tile_place_kernel(SortArgs a, Pass p, int tiles) {
    extern __shared__ uint32_t shared[];
    const int digits = 1 << p.bits;
    uint32_t* counts = shared;                  // [WARPS][digits]
    uint32_t* local = counts + WARPS * digits;  // [digits] first place in the tile
    uint32_t* shift_to = local + digits;        // [digits] place in the whole minus place in the tile
    uint32_t* keys = shift_to + digits;         // [TILE]
    uint32_t* index = keys + TILE;              // [TILE]
    __shared__ uint32_t scan[WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long begin = (long long)blockIdx.x * TILE;
    const int live = int(min((long long)TILE, a.n - begin));
    uint32_t key[ROUNDS], id[ROUNDS], rank[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int i = (warp * ROUNDS + r) * 32 + lane;
        const long long at = begin + min(i, live - 1);
        key[r] = read_key<SOURCE>(p.keys, at, uint32_t(a.bins));
        id[r] = SOURCE ? uint32_t(at) : __ldg(p.index + at);
    }
    warp_ranks(key, ROUNDS, live, p.shift, p.bits, counts, rank);
    uint32_t running = 0, running_local = 0;
    for (int base = 0; base < digits; base += THREADS) {
        const int d = base + threadIdx.x;
        uint32_t total, tile_total, c = 0, all = 0, earlier = 0;
        if (d < digits) {
#pragma unroll
            for (int w = 0; w < WARPS; ++w) c += counts[w * digits + d];
            if (tiles) {
#pragma unroll 16
                for (int t = 0; t < tiles; ++t) {
                    const uint32_t other = p.tiles[(long long)t * digits + d];
                    all += other;
                    earlier += t < int(blockIdx.x) ? other : 0;
                }
            } else {
                all = p.totals[d];
                earlier = p.tiles[(long long)blockIdx.x * digits + d];
            }
        }
        const uint32_t before = block_exclusive(all, scan, total);
        const uint32_t before_local = block_exclusive(c, scan, tile_total);
        if (d < digits) {
            local[d] = running_local + before_local;
            shift_to[d] = running + before + earlier - local[d];
            // one pass: the digit is the key
            if (!p.keys_out && SOURCE && a.offsets && blockIdx.x == 0 && d <= a.bins) a.offsets[d] = int(running + before);
        }
        running += total;
        running_local += tile_total;
    }
    __syncthreads();
    warp_starts(counts, digits, local);
    const bool last = !p.keys_out;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int i = (warp * ROUNDS + r) * 32 + lane;
        if (i < live) {
            const uint32_t d = (key[r] >> p.shift) & uint32_t(digits - 1), place = counts[warp * digits + d] + rank[r];
            const bool kept = key[r] < uint32_t(a.bins);
            keys[place] = key[r];
            index[place] = last && !kept ? ~id[r] : id[r];
            if (last && a.slot) a.slot[id[r]] = kept ? int(place + shift_to[d]) : ~int(place + shift_to[d]);
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int i = r * THREADS + threadIdx.x;
        if (i < live) {
            const uint32_t k = keys[i], place = i + shift_to[(k >> p.shift) & uint32_t(digits - 1)];
            if (last) {
                a.order[place] = int(index[i]);
                if (a.sorted) a.sorted[place] = k;
            } else {
                p.keys_out[place] = k;
                p.index_out[place] = index[i];
            }
        }
    }
}

// offsets[d]: lower bound of d among the sorted keys.
__global__ void __launch_bounds__(THREADS) key_offsets_kernel(const uint32_t* sorted, long long n, int bins, int* offsets) {
    const int d = blockIdx.x * THREADS + threadIdx.x;
    if (d > bins) return;
    long long lo = 0, hi = n;
    while (lo < hi) {
        const long long mid = (lo + hi) / 2;
        if (sorted[mid] < uint32_t(d)) lo = mid + 1;
        else hi = mid;
    }
    offsets[d] = int(lo);
}

__global__ void __launch_bounds__(THREADS) zero_offsets_kernel(int* offsets, int count) {
    const int d = blockIdx.x * THREADS + threadIdx.x;
    if (d < count) offsets[d] = 0;
}

int64_t padded(int64_t words) { return (words + 63) / 64 * 64; }

}  // namespace

int64_t sort_scratch_bytes(int64_t n, int bins) {
    if (n <= ONE_TILE) return 0;
    const int64_t digits = int64_t(1) << digit_bits(bins), tiles = (n + TILE - 1) / TILE;
    const int passes = pass_count(bins);
    // tile counts, totals, and for more than one pass two pair buffers and the sorted keys
    int64_t words = padded(tiles * digits) + padded(digits);
    if (passes > 1) words += (passes > 2 ? 4 : 2) * padded(n) + padded(n);
    return 4 * words;
}

void launch_sort(const SortArgs& a, cudaStream_t stream) {
    ODIE_REQUIRE(a.key_bytes == 4 || a.key_bytes == 8, "keys are int32 or int64");
    ODIE_REQUIRE(a.n >= 0 && a.n < (int64_t(1) << 31) - ONE_TILE, "0 to 2^31 - 4097 keys");
    ODIE_REQUIRE(a.bins >= 1 && a.bins < (1 << 30), "1 to 2^30 - 1 bins");
    if (a.n == 0) {
        if (a.offsets) {
            zero_offsets_kernel<<<blocks_for(a.bins + 1, THREADS), THREADS, 0, stream>>>(a.offsets, a.bins + 1);
            ODIE_CUDA(cudaGetLastError());
            note_launch();
        }
        return;
    }
    const int passes = pass_count(a.bins), bits = digit_bits(a.bins), digits = 1 << bits;
    const bool wide = a.key_bytes == 8;
    if (a.n <= ONE_TILE) {
        const size_t bytes = (size_t(WARPS + 1) * digits + (passes > 1 || a.sorted ? 2 : 1) * ONE_TILE) * 4;
        const auto kernel = wide ? sort_tile_kernel<8> : sort_tile_kernel<4>;
        if (bytes > 48 * 1024)
            ODIE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           ((WARPS + 1) * (1 << MAX_DIGIT_BITS) + 2 * ONE_TILE) * 4));
        kernel<<<1, THREADS, bytes, stream>>>(a, passes, bits);
        ODIE_CUDA(cudaGetLastError());
        note_launch();
        return;
    }
    ODIE_REQUIRE(a.scratch, "scratch is missing");
    const int tiles = int((a.n + TILE - 1) / TILE);
    uint32_t* at = static_cast<uint32_t*>(a.scratch);
    Pass p{};
    p.bits = bits;
    p.tiles = at;
    p.totals = p.tiles + padded(int64_t(tiles) * digits);
    at = p.totals + padded(digits);
    uint32_t* buffers[2][2] = {};
    SortArgs last = a;
    if (passes > 1) {
        for (int b = 0; b < (passes > 2 ? 2 : 1); ++b)
            for (int i = 0; i < 2; ++i, at += padded(a.n)) buffers[b][i] = at;
        if (!last.sorted) last.sorted = at;  // the offsets are read off the sorted keys
    }
    for (int i = 0; i < passes; ++i) {
        p.keys = i == 0 ? a.keys : buffers[(i - 1) % 2][0];
        p.index = i == 0 ? nullptr : buffers[(i - 1) % 2][1];
        p.keys_out = i + 1 < passes ? buffers[i % 2][0] : nullptr;
        p.index_out = i + 1 < passes ? buffers[i % 2][1] : nullptr;
        p.shift = i * bits;
        const auto counts = i > 0 ? tile_counts_kernel<0> : wide ? tile_counts_kernel<8> : tile_counts_kernel<4>;
        const auto place = i > 0 ? tile_place_kernel<0> : wide ? tile_place_kernel<8> : tile_place_kernel<4>;
        counts<<<tiles, THREADS, size_t(digits) * 4, stream>>>(last, p);
        if (tiles > FOLD) {
            tile_starts_kernel<<<(digits + 31) / 32, 1024, 0, stream>>>(p, tiles);
            note_launch();
        }
        const size_t bytes = (size_t(WARPS + 2) * digits + 2 * TILE) * 4;
        if (bytes > 48 * 1024)
            ODIE_CUDA(cudaFuncSetAttribute(place, cudaFuncAttributeMaxDynamicSharedMemorySize, ((WARPS + 2) * (1 << MAX_DIGIT_BITS) + 2 * TILE) * 4));
        place<<<tiles, THREADS, bytes, stream>>>(last, p, tiles > FOLD ? 0 : tiles);
        ODIE_CUDA(cudaGetLastError());
        note_launch(2);
    }
    if (passes > 1 && a.offsets) {
        key_offsets_kernel<<<blocks_for(a.bins + 1, THREADS), THREADS, 0, stream>>>(last.sorted, a.n, a.bins, a.offsets);
        ODIE_CUDA(cudaGetLastError());
        note_launch();
    }
}

}  // namespace odie

using namespace odie;

extern "C" int64_t odie_sort_rows_scratch(int64_t n, int bins) {
    if (n < 0 || bins < 1) return 0;
    return sort_scratch_bytes(n, bins);
}

extern "C" int odie_sort_rows(const void* keys, int key_bytes, int64_t n, int bins, int32_t* order, int32_t* slot,
                              int32_t* offsets, void* scratch, uint64_t stream) {
    return guarded([&] {
        ODIE_REQUIRE(n == 0 || (keys && order && slot), "keys, order and slot are required");
        ODIE_REQUIRE(offsets, "offsets is required");
        SortArgs a;
        a.keys = keys;
        a.key_bytes = key_bytes;
        a.n = n;
        a.bins = bins;
        a.order = order;
        a.slot = slot;
        a.offsets = offsets;
        a.scratch = scratch;
        launch_sort(a, reinterpret_cast<cudaStream_t>(stream));
    });
}
