// Embedding lookup with scaling, and the dense gradient of the table (include/elx_ops.h).
//
//   y[i] = round(scale * W[index[i]])            dW[v] = round(scale * sum of dy[i] over index[i] = v)
//
// Forward is a gather: every row read and written once, 16 bytes per lane where the alignment allows.
//
// Backward sums the rows of dy that belong to one row of the table in the order of the tokens, in fp32, and rounds once.  To
// have them side by side the tokens are sorted by index: a stable radix sort of (index, position), least significant digit
// first -- in LDS by one workgroup where the tokens fit there, else by up to 64 workgroups, one launch per digit and one to
// begin with.  Then
//   sum_kernel   one workgroup per tile of 8 or 24 sorted tokens: a run of equal indices inside the tile goes straight to its
//                row, a run that reaches over an end of the tile leaves an fp32 partial row; the workgroups behind these
//                clear the rows that no token names, which a search in the sorted tokens tells them: dW is written once;
//   join_kernel  adds up the partial rows of the runs over several tiles (a frequent token), in the order of the tiles.
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
constexpr uint32_t kSmallTokens = 4096;    // sorted by one workgroup
constexpr uint32_t kGathered = 8192;       // counters of the next pass that a workgroup gathers in LDS

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
    __shared__ uint32_t base[kMaxBins];
    __shared__ uint16_t in_wave[kSortWaves][kMaxBins];
    __shared__ uint32_t wave_total[kSortWaves];
    __shared__ uint32_t gathered[kGathered];
    const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;

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
        for (int w = 0; w < kSortWaves; ++w) in_wave[w][threadIdx.x] = 0;
        if (clear) clear[blockIdx.x * bins + threadIdx.x] = 0;
    }
    const uint32_t smaller = digits_before(total, wave_total);
    if (threadIdx.x < bins) base[threadIdx.x] = smaller + before;
    // where they fit, the next pass's counts are gathered in LDS: a frequent token would have a thousand threads add to one
    // word of memory
    const uint32_t counters = next ? gridDim.x * bins : 0;
    const bool gather = counters <= kGathered;
    if (gather)
        for (uint32_t d = threadIdx.x; d < counters; d += kSortThreads) gathered[d] = 0;
    __syncthreads();

    const uint64_t begin = (uint64_t)blockIdx.x * per_block;
    for (uint32_t round = 0; round < per_block; round += kSortThreads) {
        const uint64_t i = begin + round + threadIdx.x;
        const bool live = i < n;
        const uint32_t key = live ? key_at(in, i) : 0;
        const uint32_t digit = (key >> shift) & (bins - 1);
        const uint64_t same = lanes_with(digit, bits, live);
        const uint32_t rank = __builtin_popcountll(same & ((1ull << lane) - 1));
        if (live && rank == 0) in_wave[wave][digit] = (uint16_t)__builtin_popcountll(same);
        __syncthreads();
        if (live) {
            uint32_t at = base[digit] + rank;
            for (uint32_t w = 0; w < wave; ++w) at += in_wave[w][digit];
            keys_out[at] = key;
            positions_out[at] = in.keys ? in.positions[i] : (uint32_t)i;
            if (next) {
                const uint32_t slot = at / per_block * bins + ((key >> (shift + bits)) & (bins - 1));
                if (gather)
                    atomicAdd(&gathered[slot], 1u);
                else
                    atomicAdd(&next[slot], 1u);
            }
        }
        __syncthreads();
        if (threadIdx.x < bins) {    // the round's tokens become earlier ones
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
    if (gather)
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

// Tokens of a tile.  Few tokens: short tiles, the launch lasts as long as its longest chain of them (1021 tokens of a
// 50257 x 768 fp16 table: 25 us with 8, 29 with 16, 33 with 24).  Many: long ones, every end of a tile that cuts a run costs
// two fp32 rows (16384 tokens of 50272 x 2048 bf16: 68 us with 24, 71 with 16, 76 with 8; 75 with 32, whose rows take too
// many registers).
constexpr uint32_t kTileFew = 8, kTileMany = 24;
constexpr uint32_t kFewTokens = kSmallTokens;
constexpr int kSumThreads = 256;

constexpr uint32_t kFillBytes = 16u << 10;    // cleared by one workgroup, about
constexpr uint32_t kFillRows = 2048;          // rows of a clearing workgroup, at most

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

// First place in keys[from, n) whose key is not `key` (all before it are).
__device__ __forceinline__ uint32_t key_run_end(const uint32_t *__restrict__ keys, uint32_t n, uint32_t from, uint32_t key) {
    return from >= n ? n : from + first_at_least(keys + from, n - from, key + 1);
}

// Clears those of the rows [row, row + count) that no token names.  A row is cleared in units of `unit` bytes.
__device__ __forceinline__ void clear_rows(const uint32_t *__restrict__ keys, uint32_t n, uint32_t row, uint32_t count, char *base,
                                           uint32_t row_bytes, uint32_t unit) {
    __shared__ uint32_t named[kFillRows / 32];
    for (uint32_t i = threadIdx.x; i < kFillRows / 32; i += kSumThreads) named[i] = 0;
    __syncthreads();
    if (threadIdx.x < kWave) {
        uint32_t at = first_at_least(keys, n, row);
        while (at < n) {
            const uint32_t key = at + threadIdx.x < n ? keys[at + threadIdx.x] : ~0u;
            if (key < row + count) atomicOr(&named[(key - row) / 32], 1u << ((key - row) % 32));
            const uint32_t top = (uint32_t)__builtin_amdgcn_readlane((int)key, kWave - 1);
            if (top >= row + count) break;
            // behind this key's run: the 64 places looked at may all be of it, and so may thousands more
            at = key_run_end(keys, n, at + kWave, top);
        }
    }
    __syncthreads();
    const uint32_t units = row_bytes / unit;
    uint32_t r = threadIdx.x / units, u = threadIdx.x % units;
    const uint32_t rows_per_turn = kSumThreads / units, units_per_turn = kSumThreads % units;
    while (r < count) {
        if (!(named[r / 32] >> (r % 32) & 1)) {
            char *to = base + (uint64_t)(row + r) * row_bytes + (uint64_t)u * unit;
            if (unit == 16)
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
    uint32_t tile_blocks, chunks, rows_per_block, row_bytes, unit;
};

template <int D, int V, uint32_t kTokens>
__global__ __launch_bounds__(kSumThreads) void sum_kernel(const uint32_t *__restrict__ keys, const uint32_t *__restrict__ positions,
                                                          uint32_t n, uint32_t vocab, const typename Elem<D>::scalar *__restrict__ dy,
                                                          uint64_t dy_stride, uint32_t cols, float scale,
                                                          typename Elem<D>::scalar *__restrict__ dtable, float *__restrict__ partials,
                                                          Clear clear) {
    typedef Row<D, V> row_t;
    if (blockIdx.x >= clear.tile_blocks) {
        const uint32_t row = (blockIdx.x - clear.tile_blocks) * clear.rows_per_block;
        const uint32_t count = vocab - row < clear.rows_per_block ? vocab - row : clear.rows_per_block;
        clear_rows(keys, n, row, count, reinterpret_cast<char *>(dtable), clear.row_bytes, clear.unit);
        return;
    }
    const uint32_t tile = blockIdx.x / clear.chunks;
    const uint32_t first = tile * kTokens;
    const uint32_t c = (blockIdx.x % clear.chunks * kSumThreads + threadIdx.x) * V;
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
        if (j < count && mine)
            rows[j] = __builtin_nontemporal_load(
                reinterpret_cast<const typename row_t::type *>(dy + (uint64_t)position_of(j) * dy_stride + c));
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

constexpr int kJoinThreads = 1024;

// One workgroup per tile whose last run starts there and goes on; `lanes` threads side by side over the columns (J each),
// the groups of lanes take the run's tiles in turn, and the groups are added up in their order.
template <int D, int J>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(const uint32_t *__restrict__ keys, uint32_t n, uint32_t vocab, uint32_t cols,
                                                            float scale, typename Elem<D>::scalar *__restrict__ dtable,
                                                            const float *__restrict__ partials, uint32_t lanes, uint32_t tokens) {
    const uint32_t first = blockIdx.x * tokens, next = first + tokens;
    if (next >= n) return;
    const uint32_t key = keys[next - 1], behind = keys[next], before = first ? keys[first - 1] : ~0u;
    const uint32_t further = next + tokens < n ? keys[next + tokens] : ~0u;    // asked for together
    if (key >= vocab || behind != key || before == key) return;    // ends here, or came in from the tile before
    // the run reaches tile `lo`; find the last that it reaches
    uint32_t lo = blockIdx.x + 1, hi = further == key ? (n + tokens - 1) / tokens - 1 : lo;
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if (keys[mid * tokens] == key)
            lo = mid;
        else
            hi = mid - 1;
    }
    __shared__ float sums[J][kJoinThreads];
    const uint32_t group = threadIdx.x / lanes, groups = kJoinThreads / lanes, lane = threadIdx.x % lanes;
    for (uint32_t c0 = 0; c0 < cols; c0 += lanes * J) {
        const uint32_t c = c0 + lane * J;
        float s[J] = {};
        if (c < cols) {
            auto add = [&](uint64_t slot) {
                float x[J];
                __builtin_memcpy(x, __builtin_assume_aligned(partials + slot * cols + c, J * 4), J * 4);
#pragma unroll
                for (int j = 0; j < J; ++j) s[j] += x[j];
            };
            if (group == 0) add((uint64_t)blockIdx.x * 2 + 1);
#pragma unroll 4
            for (uint32_t t = blockIdx.x + 1 + group; t <= lo; t += groups) add((uint64_t)t * 2);
        }
#pragma unroll
        for (int j = 0; j < J; ++j) sums[j][threadIdx.x] = s[j];
        __syncthreads();
        if (group == 0 && c < cols) {
            for (uint32_t g = 1; g < groups; ++g)
#pragma unroll
                for (int j = 0; j < J; ++j) s[j] += sums[j][g * lanes + lane];
#pragma unroll
            for (int j = 0; j < J; ++j) dtable[(uint64_t)key * cols + c + j] = Elem<D>::from_f32(s[j] * scale);
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

Shape shape_of(uint64_t n, uint64_t vocab) {
    Shape s;
    // rounds of 1024 tokens per sorting workgroup, so many that at most kMaxSortBlocks of them share the work
    const uint64_t rounds = (n + (uint64_t)kSortThreads * kMaxSortBlocks - 1) / ((uint64_t)kSortThreads * kMaxSortBlocks);
    s.per_block = (uint32_t)(rounds * kSortThreads);
    s.sort_blocks = (uint32_t)((n + s.per_block - 1) / s.per_block);
    s.tokens = n <= kFewTokens ? kTileFew : kTileMany;
    s.tiles = (uint32_t)((n + s.tokens - 1) / s.tokens);
    int all = 1;    // keys are 0 .. vocab
    while (all < 32 && (vocab >> all)) ++all;
    s.passes = (all + 9) / 10;
    s.bits = (all + s.passes - 1) / s.passes;
    return s;
}

uint64_t round256(uint64_t x) { return (x + 255) & ~255ull; }

template <int D, int V>
int launch_sums(const Shape &s, const uint32_t *keys, const uint32_t *positions, uint64_t n, uint64_t vocab, const void *dy,
                uint64_t dy_stride, uint32_t cols, float scale, void *dtable, float *partials, hipStream_t stream) {
    typedef typename Elem<D>::scalar T;
    Clear clear;
    clear.chunks = ((cols + V - 1) / V + kSumThreads - 1) / kSumThreads;
    clear.tile_blocks = s.tiles * clear.chunks;
    clear.row_bytes = cols * (uint32_t)sizeof(T);
    clear.unit = clear.row_bytes % 16 == 0 && aligned16(dtable) ? 16 : (uint32_t)sizeof(T);
    const uint32_t rows = kFillBytes / clear.row_bytes;
    clear.rows_per_block = rows < 1 ? 1 : rows > kFillRows ? kFillRows : rows;
    const uint64_t clear_blocks = (vocab + clear.rows_per_block - 1) / clear.rows_per_block;
    const dim3 grid((uint32_t)(clear.tile_blocks + clear_blocks));
    if (s.tokens == kTileFew)
        hipLaunchKernelGGL((sum_kernel<D, V, kTileFew>), grid, dim3(kSumThreads), 0, stream, keys, positions, (uint32_t)n, (uint32_t)vocab,
                           (const T *)dy, dy_stride, cols, scale, (T *)dtable, partials, clear);
    else
        hipLaunchKernelGGL((sum_kernel<D, V, kTileMany>), grid, dim3(kSumThreads), 0, stream, keys, positions, (uint32_t)n,
                           (uint32_t)vocab, (const T *)dy, dy_stride, cols, scale, (T *)dtable, partials, clear);
    if (int rc = (int)hipGetLastError()) return rc;
    if (s.tiles < 2) return 0;
    constexpr int J = V > 1 ? 4 : 1;
    const uint32_t lanes = lanes_for((cols + J - 1) / J, 256);
    hipLaunchKernelGGL((join_kernel<D, J>), dim3(s.tiles - 1), dim3(kJoinThreads), 0, stream, keys, (uint32_t)n, (uint32_t)vocab, cols,
                       scale, (T *)dtable, partials, lanes, s.tokens);
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
    const Shape s = shape_of(n, vocab);
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
    const Shape s = shape_of(n, vocab);
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
    const bool vec = aligned16(dy) && aligned16(dtable) && cols % v == 0 && dy_stride % v == 0;
    switch (dtype) {
        case ELX_F32: return vec ? launch_sums<ELX_F32, 4>(s, k, p, n, vocab, dy, dy_stride, cols, scale, dtable, partials, st) : launch_sums<ELX_F32, 1>(s, k, p, n, vocab, dy, dy_stride, cols, scale, dtable, partials, st);
        case ELX_F16: return vec ? launch_sums<ELX_F16, 8>(s, k, p, n, vocab, dy, dy_stride, cols, scale, dtable, partials, st) : launch_sums<ELX_F16, 1>(s, k, p, n, vocab, dy, dy_stride, cols, scale, dtable, partials, st);
        default: return vec ? launch_sums<ELX_BF16, 8>(s, k, p, n, vocab, dy, dy_stride, cols, scale, dtable, partials, st) : launch_sums<ELX_BF16, 1>(s, k, p, n, vocab, dy, dy_stride, cols, scale, dtable, partials, st);
    }
}

}    // extern "C"
