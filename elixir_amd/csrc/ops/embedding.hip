// Embedding lookup with scaling, and the dense gradient of the table (include/elx_ops.h).
//
//   y[i] = round(scale * W[index[i]])            dW[v] = round(scale * sum of dy[i] over index[i] = v)
//
// Forward is a gather: every row read and written once, 16 bytes per lane where the alignment allows.  16384 tokens of 2048
// bf16 columns take 19 us (127 MB: 6.6 TB/s), 8 tokens 2.5 us.
//
// Backward sums the rows of dy that belong to one row of the table in a fixed order, in fp32, and rounds once.  Few tokens take
// one launch (direct_kernel).  For more, to have the rows of an index side by side, the tokens are sorted: a stable radix sort of
// (index, position), least significant digit first -- in LDS by one workgroup where the tokens fit there, else by up to 64
// workgroups, one launch per digit and one to begin with.  Then
//   sum_kernel   a workgroup per tile of 8 or 24 sorted tokens: a run of equal indices inside the tile goes straight to its
//                row, a run that reaches over an end of the tile leaves an fp32 partial row; the workgroups behind these
//                clear the rows that no token names, which the sorted tokens tell them: dW is written once;
//   join_kernel  adds up the partial rows of the runs over several tiles (a frequent token), in a fixed order.
// 16384 tokens of a 50272 x 2048 bf16 table take 4 + 2 x 6 us of sorting, 43 of sums and clearing (277 MB, of which 208 are
// written: 6.4 TB/s) and 7 of joining; 8191 tokens of 32000 x 4096 fp32 5 + 2 x 6, 98 (646 MB) and 6.
// No atomics on values: the result is the same every time, and a token that fills the batch is summed by many workgroups.
// (Clearing dW beside the sort instead, in the idle workgroups of its launches, made the sort three times slower -- its
// chain of small reads waits behind the stores -- and wrote the touched rows twice: 89 us against 70 for 16384 tokens in a
// 50272 x 2048 bf16 table.)
#include <utility>

#include "elx_ops_device.h"

using namespace elx_ops;

namespace {

template <int D, int V>
struct Row {    // V elements of type D as one access
    typedef typename Elem<D>::scalar type;
    static __device__ __forceinline__ void load(const type &p, float (&x)[V]) { x[0] = Elem<D>::to_f32(p); }
    static __device__ __forceinline__ type store(const float (&x)[V]) { return Elem<D>::from_f32(x[0]); }
};
template <>
struct Row<ELX_F32, 4> {
    typedef f32x4 type;
    static __device__ __forceinline__ void load(const type &p, float (&x)[4]) {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = p[k];
    }
    static __device__ __forceinline__ type store(const float (&x)[4]) { return type{x[0], x[1], x[2], x[3]}; }
};
template <int D>
struct Row<D, 8> {
    typedef u16x8 type;
    static __device__ __forceinline__ void load(const type &p, float (&x)[8]) {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = Elem<D>::to_f32(p[k]);
    }
    static __device__ __forceinline__ type store(const float (&x)[8]) {
        type p;
#pragma unroll
        for (int k = 0; k < 8; ++k) p[k] = Elem<D>::from_f32(x[k]);
        return p;
    }
};

__device__ __forceinline__ int64_t index_at(const void *index, int wide, uint64_t i) {
    return wide ? reinterpret_cast<const int64_t *>(index)[i] : (int64_t) reinterpret_cast<const int32_t *>(index)[i];
}

// ---------------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------------

constexpr int kFwdThreads = 256;

// `lanes` (a power of two up to the workgroup) threads per token
template <int D, int V>
__global__ __launch_bounds__(kFwdThreads) void embed_fwd_kernel(const void *index, int wide, uint64_t n,
                                                                const typename Elem<D>::scalar *__restrict__ table, uint64_t vocab,
                                                                uint32_t cols, float scale, typename Elem<D>::scalar *__restrict__ out,
                                                                uint32_t lanes) {
    typedef Row<D, V> row_t;
    const uint64_t token = (uint64_t)blockIdx.x * (kFwdThreads / lanes) + threadIdx.x / lanes;
    if (token >= n) return;
    const int64_t v = index_at(index, wide, token);
    const bool good = v >= 0 && (uint64_t)v < vocab;    // an index outside the table reads nothing: its row is NaN
    for (uint32_t c = (threadIdx.x % lanes) * V; c < cols; c += lanes * V) {
        float x[V];
        if (good) {
            row_t::load(*reinterpret_cast<const typename row_t::type *>(table + (uint64_t)v * cols + c), x);
#pragma unroll
            for (int k = 0; k < V; ++k) x[k] *= scale;
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) x[k] = __builtin_nanf("");
        }
        __builtin_nontemporal_store(row_t::store(x), reinterpret_cast<typename row_t::type *>(out + token * cols + c));
    }
}

// ---------------------------------------------------------------------------------------------
// sort
// ---------------------------------------------------------------------------------------------

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr uint32_t kMaxBins = 1024;       // ten bits per pass
constexpr uint32_t kMaxSortBlocks = 64;
// Up to that many tokens are sorted by one workgroup in one launch (768 columns: 1021 tokens 26 us with it, 29.5 in several
// launches; 2048 tokens 30.1 and 31.2; 4096 tokens 38.4 and 33.5).
constexpr uint32_t kSmallTokens = 2048;
// Counters of the next pass that a workgroup gathers in LDS.  Added to memory one by one they cost a pass of 16384 tokens 15 us
// instead of 6: frequent tokens meet in one word.
constexpr uint32_t kGathered = 16384;

struct Keys {
    const void *index;    // first pass: the indices themselves (keys == nullptr)
    int wide;
    const uint32_t *keys, *positions;
    uint64_t vocab;
    int64_t padding;
};

// what does not enter the gradient -- padding, an index outside the table -- sorts behind everything else
__device__ __forceinline__ uint32_t key_at(const Keys &k, uint64_t i) {
    if (k.keys) return k.keys[i];
    const int64_t v = index_at(k.index, k.wide, i);
    return v < 0 || (uint64_t)v >= k.vocab || v == k.padding ? (uint32_t)k.vocab : (uint32_t)v;
}

// the 64-bit mask of the lanes that are live and have this lane's digit
__device__ __forceinline__ uint64_t lanes_with(uint32_t digit, int bits, bool live) {
    uint64_t same = __builtin_amdgcn_ballot_w64(live);
    for (int b = 0; b < bits; ++b) {
        const bool one = (digit >> b) & 1;
        const uint64_t ones = __builtin_amdgcn_ballot_w64(one);
        same &= one ? ones : ~ones;
    }
    return same;
}

// Sum of `total` over the threads before this one (one digit per thread); called by the whole workgroup, ends with a barrier
// passed by everybody who has written wave_total.
__device__ __forceinline__ uint32_t digits_before(uint32_t total, uint32_t *wave_total) {
    const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    uint32_t sum = total;    // inclusive inside the wavefront
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const uint32_t other = __shfl_up(sum, d, kWave);
        sum += lane >= (uint32_t)d ? other : 0;
    }
    if (lane == kWave - 1) wave_total[wave] = sum;
    __syncthreads();
    uint32_t earlier = 0;
    for (uint32_t w = 0; w < wave; ++w) earlier += wave_total[w];
    return earlier + sum - total;
}

// counts[block][digit] of the block's stretch of `per_block` tokens, for the first pass; `next` (as large) is cleared for
// the second
__global__ __launch_bounds__(kSortThreads) void count_kernel(Keys in, uint64_t n, uint32_t per_block, uint32_t bins,
                                                             uint32_t *__restrict__ counts, uint32_t *__restrict__ next) {
    __shared__ uint32_t bin[kMaxBins];
    for (uint32_t d = threadIdx.x; d < bins; d += kSortThreads) bin[d] = 0;
    __syncthreads();
    const uint64_t begin = (uint64_t)blockIdx.x * per_block;
    const uint64_t end = begin + per_block < n ? begin + per_block : n;
    for (uint64_t i = begin + threadIdx.x; i < end; i += kSortThreads) atomicAdd(&bin[key_at(in, i) & (bins - 1)], 1u);
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < bins; d += kSortThreads) {
        counts[blockIdx.x * bins + d] = bin[d];
        if (next) next[blockIdx.x * bins + d] = 0;
    }
}

// Moves the block's stretch to its places: for each digit the tokens of earlier digits, of earlier blocks, of earlier
// rounds of 1024 tokens, of earlier wavefronts and of earlier lanes come first.  Counts the next pass's digits on the way
// (`next`, zero before; whole numbers, so the order of the additions does not matter) and clears `clear` for the pass after
// that.
__global__ __launch_bounds__(kSortThreads) void scatter_kernel(Keys in, uint64_t n, uint32_t per_block, int shift, int bits,
                                                               const uint32_t *__restrict__ counts, uint32_t *__restrict__ next,
                                                               uint32_t *__restrict__ clear, uint32_t *__restrict__ keys_out,
                                                               uint32_t *__restrict__ positions_out) {
    const uint32_t bins = 1u << bits;
    __shared__ uint32_t base[2][kMaxBins];
    __shared__ uint16_t in_wave[2][kSortWaves][kMaxBins];
    __shared__ uint32_t wave_total[kSortWaves];
    __shared__ uint32_t gathered[kGathered];
    const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const uint64_t begin = (uint64_t)blockIdx.x * per_block + threadIdx.x;
    uint32_t key = begin < n ? key_at(in, begin) : 0;

    // one digit per thread: all its tokens, and those in earlier blocks
    uint32_t total = 0, before = 0;
    if (threadIdx.x < bins) {
        for (uint32_t b = 0; b < gridDim.x; b += 16) {    // 16 loads on their way at a time
            uint32_t c[16];
#pragma unroll
            for (uint32_t k = 0; k < 16; ++k) c[k] = b + k < gridDim.x ? counts[(b + k) * bins + threadIdx.x] : 0;
#pragma unroll
            for (uint32_t k = 0; k < 16; ++k) {
                total += c[k];
                before += b + k < blockIdx.x ? c[k] : 0;
            }
        }
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) in_wave[0][w][threadIdx.x] = 0;
        if (clear) clear[blockIdx.x * bins + threadIdx.x] = 0;
    }
    uint32_t place = digits_before(total, wave_total) + before;    // of the next token with this thread's digit
    // where they fit, the next pass's counts are gathered in LDS: a frequent token would have a thousand threads add to one
    // word of memory
    const uint32_t counters = next ? gridDim.x * bins : 0;
    const bool gather = counters <= kGathered;
    if (gather)
        for (uint32_t d = threadIdx.x; d < counters; d += kSortThreads) gathered[d] = 0;

    // two barriers a round: the tables of a round are those of the round before the last, which everybody has left
    for (uint32_t round = 0, turn = 0; round < per_block; round += kSortThreads, turn ^= 1) {
        const uint64_t i = begin + round;
        const bool live = i < n;
        const uint32_t position = !live ? 0 : in.keys ? in.positions[i] : (uint32_t)i;
        const uint32_t digit = (key >> shift) & (bins - 1);
        const uint64_t same = lanes_with(digit, bits, live);
        const uint32_t rank = __builtin_popcountll(same & ((1ull << lane) - 1));
        if (live && rank == 0) in_wave[turn][wave][digit] = (uint16_t)__builtin_popcountll(same);
        const bool more = round + kSortThreads < per_block && i + kSortThreads < n;
        const uint32_t next_key = more ? key_at(in, i + kSortThreads) : 0;    // on its way
        __syncthreads();
        if (threadIdx.x < bins) {    // counts become places
            base[turn][threadIdx.x] = place;
            uint32_t c = 0;
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) {
                const uint32_t of_wave = in_wave[turn][w][threadIdx.x];
                in_wave[turn][w][threadIdx.x] = (uint16_t)c;
                in_wave[turn ^ 1][w][threadIdx.x] = 0;
                c += of_wave;
            }
            place += c;
        }
        __syncthreads();
        if (live) {
            const uint32_t at = base[turn][digit] + in_wave[turn][wave][digit] + rank;
            keys_out[at] = key;
            positions_out[at] = position;
            if (next) {
                const uint32_t slot = at / per_block * bins + ((key >> (shift + bits)) & (bins - 1));
                if (gather)
                    atomicAdd(&gathered[slot], 1u);
                else
                    atomicAdd(&next[slot], 1u);
            }
        }
        key = next_key;
    }
    if (!gather || !next) return;
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < counters; d += kSortThreads)
        if (gathered[d]) atomicAdd(&next[d], gathered[d]);
}

// The whole sort of up to kSmallTokens tokens by one workgroup, the same steps in LDS.
__global__ __launch_bounds__(kSortThreads) void sort_small_kernel(Keys in, uint32_t n, int passes, int bits, uint32_t *__restrict__ keys_out,
                                                                  uint32_t *__restrict__ positions_out) {
    const uint32_t bins = 1u << bits;
    __shared__ uint32_t keys[2][kSmallTokens];
    __shared__ uint16_t positions[2][kSmallTokens];
    __shared__ uint32_t base[kMaxBins];
    __shared__ uint16_t in_wave[kSortWaves][kMaxBins];
    __shared__ uint32_t wave_total[kSortWaves];
    const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    for (uint32_t i = threadIdx.x; i < n; i += kSortThreads) {
        keys[0][i] = key_at(in, i);
        positions[0][i] = (uint16_t)i;
    }
    for (uint32_t d = threadIdx.x; d < bins; d += kSortThreads)
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) in_wave[w][d] = 0;
    for (int pass = 0; pass < passes; ++pass) {
        const uint32_t *from = keys[pass & 1];
        const uint16_t *from_positions = positions[pass & 1];
        const int shift = pass * bits;
        if (threadIdx.x < bins) base[threadIdx.x] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += kSortThreads) atomicAdd(&base[(from[i] >> shift) & (bins - 1)], 1u);
        __syncthreads();
        const uint32_t total = threadIdx.x < bins ? base[threadIdx.x] : 0;
        const uint32_t smaller = digits_before(total, wave_total);
        if (threadIdx.x < bins) base[threadIdx.x] = smaller;
        __syncthreads();
        for (uint32_t round = 0; round < n; round += kSortThreads) {
            const uint32_t i = round + threadIdx.x;
            const bool live = i < n;
            const uint32_t key = live ? from[i] : 0;
            const uint32_t digit = (key >> shift) & (bins - 1);
            const uint64_t same = lanes_with(digit, bits, live);
            const uint32_t rank = __builtin_popcountll(same & ((1ull << lane) - 1));
            if (live && rank == 0) in_wave[wave][digit] = (uint16_t)__builtin_popcountll(same);
            __syncthreads();
            if (live) {
                uint32_t at = base[digit] + rank;
                for (uint32_t w = 0; w < wave; ++w) at += in_wave[w][digit];
                if (pass + 1 == passes) {
                    keys_out[at] = key;
                    positions_out[at] = from_positions[i];
                } else {
                    keys[(pass + 1) & 1][at] = key;
                    positions[(pass + 1) & 1][at] = from_positions[i];
                }
            }
            __syncthreads();
            if (threadIdx.x < bins) {
                uint32_t c = 0;
#pragma unroll
                for (int w = 0; w < kSortWaves; ++w) {
                    c += in_wave[w][threadIdx.x];
                    in_wave[w][threadIdx.x] = 0;
                }
                base[threadIdx.x] += c;
            }
            __syncthreads();
        }
    }
}

// ---------------------------------------------------------------------------------------------
// sums
// ---------------------------------------------------------------------------------------------

// Tokens of a tile.  Few elements: short tiles, the launch lasts as long as its longest chain of them (768 columns of fp16:
// 1021 tokens 25 us with 8, 33 with 24; 8192 tokens 38 and 46; 16384 tokens 42 and 45).  Many: long ones, every end of a tile
// that cuts a run costs two fp32 rows (16384 x 2048 bf16: 69 us with 8, 65 with 24, 70 with 32, whose rows take too many
// registers; 8192 x 4096 fp32: 134 with 8, 119 with 24, 130 with 16).
constexpr uint32_t kTileFew = 8, kTileMany = 24;
constexpr uint64_t kFewElems = 1ull << 24;
constexpr int kSumThreads = 256;    // at most

// A thread of a clearing workgroup clears about that much: with more, the last workgroups run on alone (8192 tokens in
// 32000 x 4096 fp32: 135 us with 64 bytes, 145 with 128, 150 with 256), with less the search weighs more (16384 x 2048
// bf16: 69 us with 64, 83 with 32).
constexpr uint32_t kFillBytes = 64;
constexpr uint32_t kFillRows = 2048;      // rows of a clearing workgroup, at most
// It looks at that many tokens of its rows one by one; beyond, a search per row is shorter (16384 tokens of a table of 30 rows:
// 21 us; 69 us when all are looked at).
constexpr uint32_t kScanTokens = 1024;

// First place in keys[0, n) whose key is at least `key`: the wavefront looks at 64 places at a time.
__device__ __forceinline__ uint32_t first_at_least(const uint32_t *__restrict__ keys, uint32_t n, uint32_t key) {
    uint32_t lo = 0, hi = n;    // the place lies in [lo, hi]
    const uint32_t lane = threadIdx.x % kWave;
    while (hi > lo) {
        const uint32_t step = (hi - lo + kWave - 1) / kWave;
        const uint32_t at = lo + (lane + 1) * step - 1;    // the last place of this lane's part
        const bool small = at < hi && keys[at] < key;
        const uint32_t parts = __builtin_popcountll(__builtin_amdgcn_ballot_w64(small));    // parts that lie before it
        const uint32_t next = lo + parts * step;
        const uint32_t end = next + step - 1;    // the part's last place may be the one
        lo = next < hi ? next : hi;
        hi = end < hi ? end : hi;
        if (step == 1) break;
    }
    return lo;
}

// Whether keys[lo, hi) names `key`; the thread by itself.
__device__ __forceinline__ bool names(const uint32_t *__restrict__ keys, uint32_t lo, uint32_t hi, uint32_t key) {
    const uint32_t end = hi;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (keys[mid] < key)
            lo = mid + 1;
        else
            hi = mid;
    }
    return lo < end && keys[lo] == key;
}

// dy that fits the memory-side cache is likely to be there, left by the launch before: ordinary loads (behind a launch that wrote
// dy, 8191 x 4096 fp32: 119 us against 136 with non-temporal ones, 16384 x 2048 bf16 64 against 73, 65536 x 768 bf16 64 against
// 77); what does not streams past it (1048576 x 128 bf16: 270 us against 277).  Where dW fits beside it rows are cleared there,
// too, for its reader, the landing of the gradient: with a launch that reads dW right behind, 1021 tokens of 50257 x 768 fp16
// take 45 us against 54, 16384 of 32000 x 1024 bf16 64 against 68 (alone 20 against 19 and 46 against 43); where it does not
// fit it costs (16384 of 32000 x 4096 bf16 104 against 86).
constexpr uint64_t kCacheBytes = 256ull << 20;

// Clears those of the rows [row, row + count) that `named` does not name, in units of `unit` bytes; `keep`: in the cache.
__device__ __forceinline__ void zero_rows(const uint32_t *named, uint32_t row, uint32_t count, char *base, uint32_t row_bytes,
                                          uint32_t unit, bool keep) {
    const uint32_t threads = blockDim.x;
    const uint32_t units = row_bytes / unit;
    uint32_t r = threadIdx.x / units, u = threadIdx.x % units;
    const uint32_t rows_per_turn = threads / units, units_per_turn = threads % units;
    while (r < count) {
        if (!(named[r / 32] >> (r % 32) & 1)) {
            char *to = base + (uint64_t)(row + r) * row_bytes + (uint64_t)u * unit;
            if (unit == 16 && keep)
                *reinterpret_cast<u32x4 *>(to) = u32x4{0, 0, 0, 0};
            else if (unit == 16)
                __builtin_nontemporal_store(u32x4{0, 0, 0, 0}, reinterpret_cast<u32x4 *>(to));
            else if (unit == 4)
                *reinterpret_cast<uint32_t *>(to) = 0;
            else
                *reinterpret_cast<uint16_t *>(to) = 0;
        }
        r += rows_per_turn;
        u += units_per_turn;
        if (u >= units) {
            u -= units;
            ++r;
        }
    }
}

// Clears those of the rows [row, row + count) that no token names.
__device__ __forceinline__ void clear_rows(const uint32_t *__restrict__ keys, uint32_t n, uint32_t row, uint32_t count, char *base,
                                           uint32_t row_bytes, uint32_t unit, bool keep) {
    __shared__ uint32_t named[kFillRows / 32];
    __shared__ uint32_t bounds[2];
    const uint32_t threads = blockDim.x, wave = threadIdx.x / kWave, waves = threads / kWave;
    for (uint32_t i = threadIdx.x; i < kFillRows / 32; i += threads) named[i] = 0;
    // the tokens of these rows are keys[lo, hi): its ends by two wavefronts side by side
    if (wave == 0) {
        const uint32_t at = first_at_least(keys, n, row);
        if (threadIdx.x == 0) bounds[0] = at;
    }
    if (wave == waves - 1) {
        const uint32_t at = first_at_least(keys, n, row + count);
        if (threadIdx.x % kWave == 0) bounds[1] = at;
    }
    __syncthreads();
    const uint32_t lo = bounds[0], hi = bounds[1];
    if (hi - lo <= kScanTokens) {    // few: look at each
        for (uint32_t i = lo + threadIdx.x; i < hi; i += threads) {
            const uint32_t key = keys[i] - row;
            atomicOr(&named[key / 32], 1u << (key % 32));
        }
    } else {    // frequent tokens: look for each row
        for (uint32_t r = threadIdx.x; r < count; r += threads)
            if (names(keys, lo, hi, row + r)) atomicOr(&named[r / 32], 1u << (r % 32));
    }
    __syncthreads();
    zero_rows(named, row, count, base, row_bytes, unit, keep);
}

template <typename F, uint32_t... I>
__device__ __forceinline__ void each_of(F &f, std::integer_sequence<uint32_t, I...>) {
    (f(std::integral_constant<uint32_t, I>{}), ...);
}
// f(0), f(1) ... with the numbers as constants: an array indexed by them stays in registers
template <uint32_t N, typename F>
__device__ __forceinline__ void each(F &&f) {
    each_of(f, std::make_integer_sequence<uint32_t, N>{});
}

struct Clear {    // the workgroups behind those of the tiles
    uint32_t tile_blocks, chunks, rows_per_block, row_bytes, unit, keep;
};

template <int D, int V, uint32_t kTokens, bool STREAM>
__global__ __launch_bounds__(kSumThreads) void sum_kernel(const uint32_t *__restrict__ keys, const uint32_t *__restrict__ positions,
                                                          uint32_t n, uint32_t vocab, const typename Elem<D>::scalar *__restrict__ dy,
                                                          uint64_t dy_stride, uint32_t cols, float scale,
                                                          typename Elem<D>::scalar *__restrict__ dtable, float *__restrict__ partials,
                                                          Clear clear) {
    typedef Row<D, V> row_t;
    if (blockIdx.x >= clear.tile_blocks) {
        const uint32_t row = (blockIdx.x - clear.tile_blocks) * clear.rows_per_block;
        const uint32_t count = vocab - row < clear.rows_per_block ? vocab - row : clear.rows_per_block;
        clear_rows(keys, n, row, count, reinterpret_cast<char *>(dtable), clear.row_bytes, clear.unit, clear.keep);
        return;
    }
    const uint32_t tile = blockIdx.x / clear.chunks;
    const uint32_t first = tile * kTokens;
    const uint32_t c = (blockIdx.x % clear.chunks * blockDim.x + threadIdx.x) * V;
    const bool mine = c < cols;
    // the tile's tokens, one per lane: from here on they are read from registers
    const uint32_t lane = threadIdx.x % kWave;
    static_assert(kTokens + 2 <= kWave, "a tile, the token before it and the one behind");
    const bool there = lane <= kTokens && first + lane < n;
    const uint32_t lane_key = there ? keys[first + lane] : ~0u;    // behind the last token there is no key
    const uint32_t lane_position = there ? positions[first + lane] : 0;
    const uint32_t key_before = first ? keys[first - 1] : ~0u;
    auto key_of = [&](uint32_t i) { return (uint32_t)__builtin_amdgcn_readlane((int)lane_key, (int)i); };
    auto position_of = [&](uint32_t i) { return (uint32_t)__builtin_amdgcn_readlane((int)lane_position, (int)i); };
    // tokens that enter the gradient: the ones behind them in the tile do not
    const uint32_t count = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < kTokens && lane_key < vocab));
    if (count == 0) return;
    uint32_t key = key_of(0);
    bool starts = key_before != key;    // the run that is being summed starts in this tile
    float acc[V] = {};
    // All rows of the tile are asked for before the first is written: loads and stores retire in one order, and a load
    // behind a store would wait for memory to take the store in.
    typename row_t::type rows[kTokens];
    each<kTokens>([&](auto j) {
        if (j < count && mine) {
            const auto *from = reinterpret_cast<const typename row_t::type *>(dy + (uint64_t)position_of(j) * dy_stride + c);
            rows[j] = STREAM ? __builtin_nontemporal_load(from) : *from;
        }
    });
    each<kTokens>([&](auto j) {
        if (j >= count) return;
        float x[V];
        row_t::load(rows[j], x);
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += x[k];
        const uint32_t next = key_of(j + 1);
        const bool ends = next != key;
        if (ends || j + 1 == count) {
            if (mine) {
                if (starts && ends) {
#pragma unroll
                    for (int k = 0; k < V; ++k) acc[k] *= scale;
                    __builtin_nontemporal_store(row_t::store(acc),
                                                reinterpret_cast<typename row_t::type *>(dtable + (uint64_t)key * cols + c));
                } else {    // slot 0: the run came in from the tile before; slot 1: it starts here and goes on
                    float *out = partials + ((uint64_t)tile * 2 + (starts ? 1 : 0)) * cols + c;
#pragma unroll
                    for (int k = 0; k < V; ++k) out[k] = acc[k];
                }
            }
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] = 0.0f;
            starts = true;
        }
        key = next;
    });
}

// ---------------------------------------------------------------------------------------------
// few tokens: one launch, no sort
// ---------------------------------------------------------------------------------------------

constexpr int kDirectThreads = 256;
constexpr uint32_t kDirectLanes = 64;    // at most, side by side over the columns
// Every workgroup reads every index, and a token that fills the batch is summed by one workgroup per chunk: for few of both.
// 768 columns of fp16: 8 tokens 16 us against 21 with the sort, 512 tokens 16.6 against 24.6, 1021 tokens 19.6 against 26.0 (all
// of one index 34 against 14); 512 tokens of 4096 fp32 columns, 8192 workgroups, 109 against 109, 1021 tokens 132 against 110.
constexpr uint32_t kDirectTokens = 1024, kDirectBlocks = 4096;

// A workgroup per token (and per chunk of the columns) looks at all tokens: the one of an index's first token sums the rows of
// all of them, groups of `lanes` threads taking them in turn and added up in their order; the others have nothing to do.  The
// workgroups behind these clear the rows that no token names.
template <int D, int V>
__global__ __launch_bounds__(kDirectThreads) void direct_kernel(Keys in, uint32_t n, const typename Elem<D>::scalar *__restrict__ dy,
                                                             uint64_t dy_stride, uint32_t cols, float scale,
                                                             typename Elem<D>::scalar *__restrict__ dtable, uint32_t lanes, Clear clear) {
    typedef Row<D, V> row_t;
    typedef typename row_t::type pack_t;
    const uint32_t vocab = (uint32_t)in.vocab;
    if (blockIdx.x >= clear.tile_blocks) {
        __shared__ uint32_t named[kFillRows / 32];
        const uint32_t row = (blockIdx.x - clear.tile_blocks) * clear.rows_per_block;
        const uint32_t count = vocab - row < clear.rows_per_block ? vocab - row : clear.rows_per_block;
        for (uint32_t i = threadIdx.x; i < kFillRows / 32; i += kDirectThreads) named[i] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += kDirectThreads) {
            const uint32_t key = key_at(in, i) - row;
            if (key < count) atomicOr(&named[key / 32], 1u << (key % 32));
        }
        __syncthreads();
        zero_rows(named, row, count, reinterpret_cast<char *>(dtable), clear.row_bytes, clear.unit, clear.keep);
        return;
    }
    __shared__ uint64_t same[kDirectTokens / kWave];    // the tokens of this index
    __shared__ uint16_t token_of[kDirectTokens];        // their places
    __shared__ float sums[kDirectThreads][V];
    const uint32_t token = blockIdx.x / clear.chunks, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const uint32_t words = (n + kWave - 1) / kWave;
    const uint32_t key = key_at(in, token);
    if (key == vocab) return;    // adds nothing
    for (uint32_t w = wave; w < words; w += kDirectThreads / kWave) {
        const uint32_t i = w * kWave + lane;
        const uint64_t m = __builtin_amdgcn_ballot_w64(i < n && key_at(in, i < n ? i : 0) == key);
        if (lane == 0) same[w] = m;
    }
    __syncthreads();
    uint32_t count = 0, earlier = 0;
    for (uint32_t w = 0; w < words; ++w) {
        const uint64_t m = same[w];
        count += __builtin_popcountll(m);
        const uint64_t behind = w * kWave <= token && token < (w + 1) * kWave ? ~0ull << (token % kWave) : w * kWave > token ? ~0ull : 0;
        earlier += __builtin_popcountll(m & ~behind);
    }
    if (earlier) return;    // the workgroup of the first token sums them
    if (count > 1) {
        uint32_t rank = 0;
        for (uint32_t w = 0; w < words; ++w) {
            const uint64_t m = same[w];
            if (w % (kDirectThreads / kWave) == wave && (m >> lane & 1))
                token_of[rank + __builtin_popcountll(m & ((1ull << lane) - 1))] = (uint16_t)(w * kWave + lane);
            rank += __builtin_popcountll(m);
        }
    } else if (threadIdx.x == 0) {
        token_of[0] = (uint16_t)token;
    }
    __syncthreads();
    const uint32_t group = threadIdx.x / lanes, groups = kDirectThreads / lanes;
    const uint32_t c = (blockIdx.x % clear.chunks * kDirectLanes + threadIdx.x % lanes) * V;
    const bool mine = c < cols;
    float acc[V] = {};
    if (mine) {
        constexpr uint32_t kAhead = 8;
        for (uint32_t k = group; k < count; k += groups * kAhead) {
            pack_t rows[kAhead];
#pragma unroll
            for (uint32_t j = 0; j < kAhead; ++j)
                if (k + j * groups < count)
                    rows[j] = *reinterpret_cast<const pack_t *>(dy + (uint64_t)token_of[k + j * groups] * dy_stride + c);
#pragma unroll
            for (uint32_t j = 0; j < kAhead; ++j)
                if (k + j * groups < count) {
                    float x[V];
                    row_t::load(rows[j], x);
#pragma unroll
                    for (int i = 0; i < V; ++i) acc[i] += x[i];
                }
        }
    }
    if (groups > 1 && count > 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) sums[threadIdx.x][i] = acc[i];
        __syncthreads();
        if (group == 0)
            for (uint32_t g = 1; g < groups && g < count; ++g)
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] += sums[g * lanes + threadIdx.x][i];
    }
    if (group == 0 && mine) {
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] *= scale;
        __builtin_nontemporal_store(row_t::store(acc), reinterpret_cast<pack_t *>(dtable + (uint64_t)key * cols + c));
    }
}

constexpr int kJoinThreads = 1024;
constexpr uint32_t kJoinLanes = 16, kJoinGroups = kJoinThreads / kJoinLanes;
constexpr uint32_t kJoinAlone = 8;
static_assert(kJoinGroups == kWave, "a wavefront looks at the tiles of all groups");

// Rows of runs over several tiles.  A workgroup looks at 64 tiles and at 16 J columns.  A group of 16 lanes per tile whose last
// run starts there and goes on adds its partial rows up; a run over more than kJoinAlone further tiles is left to the whole
// workgroup: its groups take the run's tiles in turn and are added up in their order.  Narrow slices of the columns let many
// workgroups share the run of a token that fills the batch (16384 x 2048 bf16 of one token: 35 us in all, 124 with the
// whole row in one workgroup per run).
template <int D, int J>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(const uint32_t *__restrict__ keys, uint32_t n, uint32_t vocab, uint32_t cols,
                                                            float scale, typename Elem<D>::scalar *__restrict__ dtable,
                                                            const float *__restrict__ partials, uint32_t tokens, uint32_t chunks) {
    __shared__ uint32_t run_key[kJoinGroups], run_last[kJoinGroups];    // of the run that each tile begins: its key, its last tile
    __shared__ uint64_t long_runs;                                      // the tiles whose run is left to the workgroup
    __shared__ float sums[kJoinGroups][kJoinLanes * J];
    const uint32_t tile0 = blockIdx.x / chunks * kJoinGroups, c0 = blockIdx.x % chunks * (kJoinLanes * J);
    if (threadIdx.x < kWave) {
        const uint32_t tile = tile0 + threadIdx.x, next = (tile + 1) * tokens;
        uint32_t key = ~0u, last = 0;
        if (next < n) {
            // the tile's last key, the one before it and the first ones of the tiles behind it, asked for together
            const uint32_t k = keys[next - 1], before = tile ? keys[tile * tokens - 1] : ~0u;
            uint32_t ahead[kJoinAlone + 1];
#pragma unroll
            for (uint32_t i = 0; i <= kJoinAlone; ++i) {
                const uint32_t at = next + i * tokens;
                ahead[i] = at < n ? keys[at] : ~0u;
            }
            uint32_t reach = 0;    // tiles behind this one that start with the key: keys are sorted, so they come first
#pragma unroll
            for (uint32_t i = 0; i <= kJoinAlone; ++i) reach += ahead[i] == k ? 1 : 0;
            if (k < vocab && before != k && reach) {
                key = k;
                last = tile + reach;
                uint32_t hi = reach > kJoinAlone ? (n + tokens - 1) / tokens - 1 : last;    // beyond what has been looked at
                while (last < hi) {
                    const uint32_t mid = (last + hi + 1) / 2;
                    if (keys[mid * tokens] == k)
                        last = mid;
                    else
                        hi = mid - 1;
                }
            }
        }
        run_key[threadIdx.x] = key;
        run_last[threadIdx.x] = last;
        const uint64_t far = __builtin_amdgcn_ballot_w64(key != ~0u && last - tile > kJoinAlone);
        if (threadIdx.x == 0) long_runs = far;
    }
    __syncthreads();
    const uint32_t group = threadIdx.x / kJoinLanes, lane = threadIdx.x % kJoinLanes, c = c0 + lane * J;
    const bool mine = c < cols;
    auto add = [&](uint64_t slot, float (&s)[J]) {
        float x[J];
        __builtin_memcpy(x, __builtin_assume_aligned(partials + slot * cols + c, J * 4), J * 4);
#pragma unroll
        for (int j = 0; j < J; ++j) s[j] += x[j];
    };
    {
        const uint32_t key = run_key[group], tile = tile0 + group, last = run_last[group];
        if (mine && key != ~0u && last - tile <= kJoinAlone) {
            float s[J] = {};
            add((uint64_t)tile * 2 + 1, s);
#pragma unroll 4
            for (uint32_t t = tile + 1; t <= last; ++t) add((uint64_t)t * 2, s);
#pragma unroll
            for (int j = 0; j < J; ++j) dtable[(uint64_t)key * cols + c + j] = Elem<D>::from_f32(s[j] * scale);
        }
    }
    for (uint64_t left = long_runs; left; left &= left - 1) {
        const uint32_t g = __builtin_ctzll(left), key = run_key[g], tile = tile0 + g, last = run_last[g];
        float s[J] = {};
        if (mine) {
            if (group == 0) add((uint64_t)tile * 2 + 1, s);
#pragma unroll 8
            for (uint32_t t = tile + 1 + group; t <= last; t += kJoinGroups) add((uint64_t)t * 2, s);
        }
#pragma unroll
        for (int j = 0; j < J; ++j) sums[group][lane * J + j] = s[j];
        __syncthreads();
        if (threadIdx.x < kJoinLanes * J && c0 + threadIdx.x < cols) {
            float all = 0.0f;
#pragma unroll 16
            for (uint32_t i = 0; i < kJoinGroups; ++i) all += sums[i][threadIdx.x];
            dtable[(uint64_t)key * cols + c0 + threadIdx.x] = Elem<D>::from_f32(all * scale);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------

constexpr uint64_t kMaxTokens = 1ull << 26, kMaxVocab = 1ull << 30;    // a launch has at most 2^32 threads
constexpr uint32_t kMaxCols = 1u << 20;
constexpr uint64_t kMaxElems = 1ull << 34;    // of dy and of the table: fewer than 2^24 workgroups of 256 in the sum

uint32_t lanes_for(uint32_t accesses, uint32_t most) {
    uint32_t l = 1;
    while (l < accesses && l < most) l <<= 1;
    return l;
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

template <int D, int V>
int launch_fwd(const void *index, int wide, uint64_t n, const void *table, uint64_t vocab, uint32_t cols, float scale, void *out,
               hipStream_t stream) {
    typedef typename Elem<D>::scalar T;
    const uint32_t lanes = lanes_for((cols + V - 1) / V, kFwdThreads), tokens = kFwdThreads / lanes;
    hipLaunchKernelGGL((embed_fwd_kernel<D, V>), dim3((uint32_t)((n + tokens - 1) / tokens)), dim3(kFwdThreads), 0, stream, index, wide,
                       n, (const T *)table, vocab, cols, scale, (T *)out, lanes);
    return (int)hipGetLastError();
}

struct Shape {
    uint32_t per_block, sort_blocks, tokens, tiles;    // tokens of a tile, tiles
    int passes, bits;
};

Shape shape_of(uint64_t n, uint64_t vocab, uint32_t cols) {
    Shape s;
    int all = 1;    // keys are 0 .. vocab
    while (all < 32 && (vocab >> all)) ++all;
    s.passes = (all + 9) / 10;
    s.bits = (all + s.passes - 1) / s.passes;
    // Rounds of 1024 tokens per sorting workgroup, so many that at most kMaxSortBlocks of them share the work -- half of them
    // where their counters of the next pass then fit LDS (131072 tokens of 128256 rows: 97 us with half, 108 with all; a
    // quarter costs more than it gains, 1000000 rows: 140 us, 124 with all).
    const uint64_t most = s.passes > 1 && (kMaxSortBlocks << s.bits) == 2 * kGathered ? kMaxSortBlocks / 2 : kMaxSortBlocks;
    const uint64_t rounds = (n + kSortThreads * most - 1) / (kSortThreads * most);
    s.per_block = (uint32_t)(rounds * kSortThreads);
    s.sort_blocks = (uint32_t)((n + s.per_block - 1) / s.per_block);
    s.tokens = n * cols <= kFewElems ? kTileFew : kTileMany;
    s.tiles = (uint32_t)((n + s.tokens - 1) / s.tokens);
    return s;
}

uint64_t round256(uint64_t x) { return (x + 255) & ~255ull; }

// the clearing workgroups of `threads` threads behind `tile_blocks` others; returns how many
template <int D>
uint64_t plan_clear(Clear *clear, uint64_t n, uint64_t vocab, uint32_t cols, const void *dtable, uint32_t threads) {
    const uint32_t es = elem_size(D);
    clear->row_bytes = cols * es;
    clear->unit = clear->row_bytes % 16 == 0 && aligned16(dtable) ? 16 : es;
    clear->keep = (n + vocab) * clear->row_bytes <= kCacheBytes;
    const uint32_t rows = kFillBytes * threads / clear->row_bytes;
    clear->rows_per_block = rows < 1 ? 1 : rows > kFillRows ? kFillRows : rows;
    return (vocab + clear->rows_per_block - 1) / clear->rows_per_block;
}

struct Grad {
    const void *dy;
    uint64_t n, vocab, dy_stride;
    uint32_t cols;
    float scale;
    void *dtable;
    hipStream_t stream;
};

template <int V>
uint32_t direct_chunks(uint32_t cols) {
    return ((cols + V - 1) / V + kDirectLanes - 1) / kDirectLanes;
}

template <int D, int V>
int launch_direct(const Keys &in, const Grad &a) {
    typedef typename Elem<D>::scalar T;
    Clear clear;
    clear.chunks = direct_chunks<V>(a.cols);
    clear.tile_blocks = (uint32_t)a.n * clear.chunks;
    const uint64_t clear_blocks = plan_clear<D>(&clear, a.n, a.vocab, a.cols, a.dtable, kDirectThreads);
    hipLaunchKernelGGL((direct_kernel<D, V>), dim3((uint32_t)(clear.tile_blocks + clear_blocks)), dim3(kDirectThreads), 0, a.stream, in,
                       (uint32_t)a.n, (const T *)a.dy, a.dy_stride, a.cols, a.scale, (T *)a.dtable,
                       lanes_for((a.cols + V - 1) / V, kDirectLanes), clear);
    return (int)hipGetLastError();
}

template <int D, int V>
int launch_sums(const Shape &s, const uint32_t *keys, const uint32_t *positions, float *partials, const Grad &a) {
    typedef typename Elem<D>::scalar T;
    const uint32_t accesses = (a.cols + V - 1) / V;
    Clear clear;
    clear.chunks = (accesses + kSumThreads - 1) / kSumThreads;
    clear.tile_blocks = s.tiles * clear.chunks;
    // whole wavefronts, no more than the columns need: idle ones would take the place of other tiles
    const dim3 threads(((accesses + clear.chunks - 1) / clear.chunks + kWave - 1) / kWave * kWave);
    const uint64_t clear_blocks = plan_clear<D>(&clear, a.n, a.vocab, a.cols, a.dtable, threads.x);
    const dim3 grid((uint32_t)(clear.tile_blocks + clear_blocks));
    const uint32_t n = (uint32_t)a.n, vocab = (uint32_t)a.vocab;
    auto kernel = sum_kernel<D, V, kTileFew, false>;    // kFewElems elements fit the cache
    if (s.tokens == kTileMany)
        kernel = a.n * a.cols * sizeof(T) > kCacheBytes ? sum_kernel<D, V, kTileMany, true> : sum_kernel<D, V, kTileMany, false>;
    hipLaunchKernelGGL(kernel, grid, threads, 0, a.stream, keys, positions, n, vocab, (const T *)a.dy, a.dy_stride, a.cols, a.scale,
                       (T *)a.dtable, partials, clear);
    if (int rc = (int)hipGetLastError()) return rc;
    if (s.tiles < 2) return 0;
    constexpr int J = V > 1 ? 4 : 1;
    const uint32_t chunks = (a.cols + kJoinLanes * J - 1) / (kJoinLanes * J);
    hipLaunchKernelGGL((join_kernel<D, J>), dim3((s.tiles - 1 + kJoinGroups - 1) / kJoinGroups * chunks), dim3(kJoinThreads), 0, a.stream,
                       keys, n, vocab, a.cols, a.scale, (T *)a.dtable, partials, s.tokens, chunks);
    return (int)hipGetLastError();
}

}    // namespace

extern "C" {

int elx_embedding_fwd(const void *index, int index_bytes, uint64_t n, const void *table, uint64_t vocab, uint32_t cols, float scale,
                      void *out, int dtype, void *stream) {
    if (!index || !table || !out) return ELX_E_NULL;
    if (!is_float_code(dtype) || (index_bytes != 4 && index_bytes != 8)) return ELX_E_DTYPE;
    if (n == 0 || n > kMaxTokens || vocab == 0 || vocab > kMaxVocab || cols == 0 || cols > kMaxCols) return ELX_E_SIZE;
    const uint32_t es = elem_size(dtype), v = 16 / es;
    if (((uintptr_t)index & (index_bytes - 1)) || (((uintptr_t)table | (uintptr_t)out) & (es - 1))) return ELX_E_ALIGN;
    const bool vec = aligned16(table) && aligned16(out) && cols % v == 0;
    const int wide = index_bytes == 8;
    // a launch has at most 2^32 threads: tokens in pieces
    for (uint64_t i = 0; i < n; i += 1ull << 23) {
        const uint64_t m = n - i < (1ull << 23) ? n - i : 1ull << 23;
        const void *at = (const char *)index + i * index_bytes;
        void *to = (char *)out + i * cols * es;
        hipStream_t st = (hipStream_t)stream;
        int rc;
        switch (dtype) {
            case ELX_F32: rc = vec ? launch_fwd<ELX_F32, 4>(at, wide, m, table, vocab, cols, scale, to, st) : launch_fwd<ELX_F32, 1>(at, wide, m, table, vocab, cols, scale, to, st); break;
            case ELX_F16: rc = vec ? launch_fwd<ELX_F16, 8>(at, wide, m, table, vocab, cols, scale, to, st) : launch_fwd<ELX_F16, 1>(at, wide, m, table, vocab, cols, scale, to, st); break;
            default: rc = vec ? launch_fwd<ELX_BF16, 8>(at, wide, m, table, vocab, cols, scale, to, st) : launch_fwd<ELX_BF16, 1>(at, wide, m, table, vocab, cols, scale, to, st);
        }
        if (rc) return rc;
    }
    return 0;
}

uint64_t elx_embedding_bwd_workspace(uint64_t n, uint64_t vocab, uint32_t cols) {
    if (n == 0 || n > kMaxTokens || vocab == 0 || vocab > kMaxVocab || cols == 0 || cols > kMaxCols || n * cols > kMaxElems) return 0;
    const Shape s = shape_of(n, vocab, cols);
    return 4 * round256(4 * n) + 3 * round256((uint64_t)s.sort_blocks * kMaxBins * 4) + round256((uint64_t)s.tiles * 2 * cols * 4);
}

int elx_embedding_bwd(const void *index, int index_bytes, uint64_t n, const void *dy, uint64_t dy_stride, void *dtable, uint64_t vocab,
                      uint32_t cols, float scale, int64_t padding, void *workspace, uint64_t workspace_bytes, int dtype, void *stream) {
    if (!index || !dy || !dtable || !workspace) return ELX_E_NULL;
    if (!is_float_code(dtype) || (index_bytes != 4 && index_bytes != 8)) return ELX_E_DTYPE;
    if (n == 0 || n > kMaxTokens || vocab == 0 || vocab > kMaxVocab || cols == 0 || cols > kMaxCols) return ELX_E_SIZE;
    if (n * cols > kMaxElems || vocab * cols > kMaxElems) return ELX_E_SIZE;
    if ((dy_stride < cols && n > 1) || dy_stride > (1ull << 36)) return ELX_E_RANGE;
    if (workspace_bytes < elx_embedding_bwd_workspace(n, vocab, cols)) return ELX_E_SIZE;
    const uint32_t es = elem_size(dtype), v = 16 / es;
    if (((uintptr_t)index & (index_bytes - 1)) || (((uintptr_t)dy | (uintptr_t)dtable) & (es - 1)) || ((uintptr_t)workspace & 15u))
        return ELX_E_ALIGN;
    const Grad grad = {dy, n, vocab, dy_stride, cols, scale, dtable, (hipStream_t)stream};
    const bool vec = aligned16(dy) && aligned16(dtable) && cols % v == 0 && dy_stride % v == 0;
    const uint64_t chunks = !vec ? direct_chunks<1>(cols) : es == 4 ? direct_chunks<4>(cols) : direct_chunks<8>(cols);
    if (n <= kDirectTokens && n * chunks <= kDirectBlocks) {
        const Keys in = {index, index_bytes == 8, nullptr, nullptr, vocab, padding};
        switch (dtype) {
            case ELX_F32: return vec ? launch_direct<ELX_F32, 4>(in, grad) : launch_direct<ELX_F32, 1>(in, grad);
            case ELX_F16: return vec ? launch_direct<ELX_F16, 8>(in, grad) : launch_direct<ELX_F16, 1>(in, grad);
            default: return vec ? launch_direct<ELX_BF16, 8>(in, grad) : launch_direct<ELX_BF16, 1>(in, grad);
        }
    }
    const Shape s = shape_of(n, vocab, cols);
    char *at = (char *)workspace;
    uint32_t *keys[2], *positions[2];
    for (int i = 0; i < 2; ++i) {
        keys[i] = (uint32_t *)at;
        at += round256(4 * n);
        positions[i] = (uint32_t *)at;
        at += round256(4 * n);
    }
    uint32_t *counts[3];    // of this pass, of the next, and of the one after that
    for (int i = 0; i < 3; ++i) {
        counts[i] = (uint32_t *)at;
        at += round256((uint64_t)s.sort_blocks * kMaxBins * 4);
    }
    float *partials = (float *)at;

    hipStream_t st = (hipStream_t)stream;
    if (n <= kSmallTokens) {
        const Keys in = {index, index_bytes == 8, nullptr, nullptr, vocab, padding};
        hipLaunchKernelGGL(sort_small_kernel, dim3(1), dim3(kSortThreads), 0, st, in, (uint32_t)n, s.passes, s.bits,
                           keys[(s.passes - 1) & 1], positions[(s.passes - 1) & 1]);
        if (int rc = (int)hipGetLastError()) return rc;
    } else {
        for (int pass = 0; pass < s.passes; ++pass) {
            const Keys in = {index, index_bytes == 8, pass ? keys[(pass - 1) & 1] : nullptr, pass ? positions[(pass - 1) & 1] : nullptr,
                             vocab, padding};
            const bool more = pass + 1 < s.passes, yet_more = pass + 2 < s.passes;
            if (pass == 0) {
                hipLaunchKernelGGL(count_kernel, dim3(s.sort_blocks), dim3(kSortThreads), 0, st, in, n, s.per_block, 1u << s.bits, counts[0],
                                   more ? counts[1] : nullptr);
                if (int rc = (int)hipGetLastError()) return rc;
            }
            hipLaunchKernelGGL(scatter_kernel, dim3(s.sort_blocks), dim3(kSortThreads), 0, st, in, n, s.per_block, pass * s.bits, s.bits,
                               counts[pass % 3], more ? counts[(pass + 1) % 3] : nullptr, yet_more ? counts[(pass + 2) % 3] : nullptr,
                               keys[pass & 1], positions[pass & 1]);
            if (int rc = (int)hipGetLastError()) return rc;
        }
    }
    const uint32_t *k = keys[(s.passes - 1) & 1], *p = positions[(s.passes - 1) & 1];
    switch (dtype) {
        case ELX_F32: return vec ? launch_sums<ELX_F32, 4>(s, k, p, partials, grad) : launch_sums<ELX_F32, 1>(s, k, p, partials, grad);
        case ELX_F16: return vec ? launch_sums<ELX_F16, 8>(s, k, p, partials, grad) : launch_sums<ELX_F16, 1>(s, k, p, partials, grad);
        default: return vec ? launch_sums<ELX_BF16, 8>(s, k, p, partials, grad) : launch_sums<ELX_BF16, 1>(s, k, p, partials, grad);
    }
}

}    // extern "C"
