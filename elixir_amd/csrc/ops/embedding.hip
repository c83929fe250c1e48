// Embedding lookup with scaling, and the dense gradient of the table (include/elx_ops.h).
//
//   y[i] = round(scale * W[index[i]])            dW[v] = round(scale * sum of dy[i] over index[i] = v)
//
// Forward is a gather: every row read and written once, 16 bytes per lane where the alignment allows.
//
// Backward sums the rows of dy that belong to one row of the table in the order of the tokens, in fp32, and rounds once.  To
// have them side by side the tokens are sorted by index: a stable radix sort of (index, position), least significant digit
// first, in launches whose few sorting workgroups leave most of the chip idle -- the other workgroups of the same launches
// clear dW meanwhile.  Then
//   sum_kernel   one workgroup per tile of 32 sorted tokens: a run of equal indices inside the tile goes straight to its
//                row, a run that reaches over an end of the tile leaves an fp32 partial row;
//   join_kernel  adds up the partial rows of the runs over several tiles (a frequent token), in the order of the tiles.
// No atomics on values: the result is the same every time, and a token that fills the batch is summed by many workgroups.
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
constexpr uint32_t kFillBytes = 256u << 10;    // cleared by one workgroup

struct Fill {    // the part of dW that a launch clears with the workgroups behind its sorting ones
    char *base;
    uint64_t bytes;
    uint32_t unit;    // 16, or the element size of a table that is not 16-byte aligned
};

__device__ __forceinline__ void fill_part(const Fill &f, uint32_t block) {
    const uint64_t begin = (uint64_t)block * kFillBytes;
    if (begin >= f.bytes) return;
    const uint32_t bytes = f.bytes - begin < kFillBytes ? (uint32_t)(f.bytes - begin) : kFillBytes;
    char *at = f.base + begin;
    if (f.unit == 16) {
        const uint32_t whole = bytes & ~15u;
        for (uint32_t i = threadIdx.x * 16; i < whole; i += kSortThreads * 16)
            __builtin_nontemporal_store(u32x4{0, 0, 0, 0}, reinterpret_cast<u32x4 *>(at + i));
        for (uint32_t i = whole + threadIdx.x * 2; i < bytes; i += kSortThreads * 2) *reinterpret_cast<uint16_t *>(at + i) = 0;
    } else {
        for (uint32_t i = threadIdx.x * 2; i < bytes; i += kSortThreads * 2) *reinterpret_cast<uint16_t *>(at + i) = 0;
    }
}

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

// counts[block][digit] of the block's stretch of `per_block` tokens
__global__ __launch_bounds__(kSortThreads) void count_kernel(Keys in, uint64_t n, uint32_t per_block, uint32_t sort_blocks, int shift,
                                                             uint32_t bins, uint32_t *__restrict__ counts, Fill fill) {
    if (blockIdx.x >= sort_blocks) {
        fill_part(fill, blockIdx.x - sort_blocks);
        return;
    }
    __shared__ uint32_t bin[kMaxBins];
    for (uint32_t d = threadIdx.x; d < bins; d += kSortThreads) bin[d] = 0;
    __syncthreads();
    const uint64_t begin = (uint64_t)blockIdx.x * per_block;
    const uint64_t end = begin + per_block < n ? begin + per_block : n;
    for (uint64_t i = begin + threadIdx.x; i < end; i += kSortThreads) atomicAdd(&bin[(key_at(in, i) >> shift) & (bins - 1)], 1u);
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < bins; d += kSortThreads) counts[blockIdx.x * bins + d] = bin[d];
}

// Moves the block's stretch to its places: for each digit the tokens of earlier digits, of earlier blocks, of earlier
// rounds of 1024 tokens, of earlier wavefronts and of earlier lanes come first.
__global__ __launch_bounds__(kSortThreads) void scatter_kernel(Keys in, uint64_t n, uint32_t per_block, uint32_t sort_blocks, int shift,
                                                               int bits, const uint32_t *__restrict__ counts,
                                                               uint32_t *__restrict__ keys_out, uint32_t *__restrict__ positions_out,
                                                               Fill fill) {
    if (blockIdx.x >= sort_blocks) {
        fill_part(fill, blockIdx.x - sort_blocks);
        return;
    }
    const uint32_t bins = 1u << bits;
    __shared__ uint32_t base[kMaxBins];
    __shared__ uint16_t in_wave[kSortWaves][kMaxBins];
    __shared__ uint32_t wave_total[kSortWaves];
    const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;

    // one digit per thread: all its tokens, and those in earlier blocks
    uint32_t total = 0, before = 0;
    if (threadIdx.x < bins) {
        for (uint32_t b = 0; b < sort_blocks; ++b) {
            const uint32_t c = counts[b * bins + threadIdx.x];
            total += c;
            before += b < blockIdx.x ? c : 0;
        }
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) in_wave[w][threadIdx.x] = 0;
    }
    uint32_t sum = total;    // inclusive sum over the digits of the wavefront
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const uint32_t other = __shfl_up(sum, d, kWave);
        sum += lane >= (uint32_t)d ? other : 0;
    }
    if (lane == kWave - 1) wave_total[wave] = sum;
    __syncthreads();
    uint32_t earlier = 0;
    for (uint32_t w = 0; w < wave; ++w) earlier += wave_total[w];
    if (threadIdx.x < bins) base[threadIdx.x] = earlier + sum - total + before;
    __syncthreads();

    const uint64_t begin = (uint64_t)blockIdx.x * per_block;
    for (uint32_t round = 0; round < per_block; round += kSortThreads) {
        const uint64_t i = begin + round + threadIdx.x;
        const bool live = i < n;
        const uint32_t key = live ? key_at(in, i) : 0;
        const uint32_t digit = (key >> shift) & (bins - 1);
        uint64_t same = __builtin_amdgcn_ballot_w64(live);    // lanes with this lane's digit
        for (int b = 0; b < bits; ++b) {
            const bool one = (digit >> b) & 1;
            const uint64_t ones = __builtin_amdgcn_ballot_w64(one);
            same &= one ? ones : ~ones;
        }
        const uint32_t rank = __builtin_popcountll(same & ((1ull << lane) - 1));
        if (live && rank == 0) in_wave[wave][digit] = (uint16_t)__builtin_popcountll(same);
        __syncthreads();
        if (live) {
            uint32_t at = base[digit] + rank;
            for (uint32_t w = 0; w < wave; ++w) at += in_wave[w][digit];
            keys_out[at] = key;
            positions_out[at] = in.keys ? in.positions[i] : (uint32_t)i;
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
}

// ---------------------------------------------------------------------------------------------
// sums
// ---------------------------------------------------------------------------------------------

constexpr uint32_t kTokens = 32;    // of one tile
constexpr int kAhead = 8;           // rows of dy in flight per lane
constexpr int kSumThreads = 256;

template <int D, int V>
__global__ __launch_bounds__(kSumThreads) void sum_kernel(const uint32_t *__restrict__ keys, const uint32_t *__restrict__ positions,
                                                          uint32_t n, uint32_t vocab, const typename Elem<D>::scalar *__restrict__ dy,
                                                          uint64_t dy_stride, uint32_t cols, float scale,
                                                          typename Elem<D>::scalar *__restrict__ dtable, float *__restrict__ partials) {
    typedef Row<D, V> row_t;
    const uint32_t first = blockIdx.x * kTokens;
    const uint32_t last = first + kTokens < n ? first + kTokens : n;    // one behind the tile's last token
    const uint32_t c = (blockIdx.y * blockDim.x + threadIdx.x) * V;
    const bool mine = c < cols;
    uint32_t key = keys[first];
    if (key >= vocab) return;
    bool starts = first == 0 || keys[first - 1] != key;    // the run that is being summed starts in this tile
    float acc[V] = {};
    for (uint32_t j = first; j < last && key < vocab; j += kAhead) {
        typename row_t::type rows[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
            if (j + a < last && keys[j + a] < vocab && mine)
                rows[a] = __builtin_nontemporal_load(
                    reinterpret_cast<const typename row_t::type *>(dy + (uint64_t)positions[j + a] * dy_stride + c));
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            if (j + a >= last || key >= vocab) break;
            float x[V];
            row_t::load(rows[a], x);
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] += x[k];
            const uint32_t next = j + a + 1 < n ? keys[j + a + 1] : ~0u;
            const bool ends = next != key;
            if (ends || j + a + 1 == last) {
                if (mine) {
                    if (starts && ends) {
#pragma unroll
                        for (int k = 0; k < V; ++k) acc[k] *= scale;
                        *reinterpret_cast<typename row_t::type *>(dtable + (uint64_t)key * cols + c) = row_t::store(acc);
                    } else {    // slot 0: the run came in from the tile before; slot 1: it starts here and goes on
                        float *out = partials + ((uint64_t)blockIdx.x * 2 + (starts ? 1 : 0)) * cols + c;
#pragma unroll
                        for (int k = 0; k < V; ++k) out[k] = acc[k];
                    }
                }
#pragma unroll
                for (int k = 0; k < V; ++k) acc[k] = 0.0f;
                starts = true;
            }
            key = next;
        }
    }
}

constexpr int kJoinThreads = 1024;

// One workgroup per tile whose last run starts there and goes on; `lanes` threads side by side over the columns, the
// groups of lanes take the run's tiles in turn, and the groups are added up in their order.
template <int D>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(const uint32_t *__restrict__ keys, uint32_t n, uint32_t vocab, uint32_t cols,
                                                            float scale, typename Elem<D>::scalar *__restrict__ dtable,
                                                            const float *__restrict__ partials, uint32_t lanes) {
    const uint32_t first = blockIdx.x * kTokens, next = first + kTokens;
    if (next >= n) return;
    const uint32_t key = keys[next - 1];
    if (key >= vocab || keys[next] != key) return;
    if (keys[first] == key && first > 0 && keys[first - 1] == key) return;    // it came in from the tile before
    // the run's last tile
    uint32_t lo = blockIdx.x + 1, hi = (n + kTokens - 1) / kTokens - 1;    // the run reaches `lo`; find the last it reaches
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if (keys[mid * kTokens] == key)
            lo = mid;
        else
            hi = mid - 1;
    }
    __shared__ float sums[kJoinThreads];
    const uint32_t group = threadIdx.x / lanes, groups = kJoinThreads / lanes, lane = threadIdx.x % lanes;
    const uint32_t c = blockIdx.y * lanes + lane;
    float s = 0.0f;
    if (c < cols) {
        if (group == 0) s = partials[((uint64_t)blockIdx.x * 2 + 1) * cols + c];
        for (uint32_t t = blockIdx.x + 1 + group; t <= lo; t += groups) s += partials[(uint64_t)t * 2 * cols + c];
    }
    sums[threadIdx.x] = s;
    __syncthreads();
    if (group == 0 && c < cols) {
        for (uint32_t g = 1; g < groups; ++g) s += sums[g * lanes + lane];
        dtable[(uint64_t)key * cols + c] = Elem<D>::from_f32(s * scale);
    }
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------

constexpr uint64_t kMaxTokens = 1ull << 26, kMaxVocab = 1ull << 30;    // a launch has at most 2^32 threads
constexpr uint32_t kMaxCols = 1u << 20;

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
    uint32_t per_block, sort_blocks, tiles;
    int passes, bits;
};

Shape shape_of(uint64_t n, uint64_t vocab) {
    Shape s;
    // rounds of 1024 tokens per sorting workgroup, so many that at most kMaxSortBlocks of them share the work
    const uint64_t rounds = (n + (uint64_t)kSortThreads * kMaxSortBlocks - 1) / ((uint64_t)kSortThreads * kMaxSortBlocks);
    s.per_block = (uint32_t)(rounds * kSortThreads);
    s.sort_blocks = (uint32_t)((n + s.per_block - 1) / s.per_block);
    s.tiles = (uint32_t)((n + kTokens - 1) / kTokens);
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
    const uint32_t accesses = (cols + V - 1) / V;
    const uint32_t threads = accesses >= kSumThreads ? kSumThreads : (accesses + kWave - 1) / kWave * kWave;
    hipLaunchKernelGGL((sum_kernel<D, V>), dim3(s.tiles, (accesses + threads - 1) / threads), dim3(threads), 0, stream, keys, positions,
                       (uint32_t)n, (uint32_t)vocab, (const T *)dy, dy_stride, cols, scale, (T *)dtable, partials);
    if (int rc = (int)hipGetLastError()) return rc;
    if (s.tiles < 2) return 0;
    const uint32_t lanes = lanes_for(cols, 256);
    hipLaunchKernelGGL((join_kernel<D>), dim3(s.tiles - 1, (cols + lanes - 1) / lanes), dim3(kJoinThreads), 0, stream, keys, (uint32_t)n,
                       (uint32_t)vocab, cols, scale, (T *)dtable, partials, lanes);
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
    if (n == 0 || n > kMaxTokens || vocab == 0 || vocab > kMaxVocab || cols == 0 || cols > kMaxCols) return 0;
    const Shape s = shape_of(n, vocab);
    return 4 * round256(4 * n) + round256((uint64_t)s.sort_blocks * kMaxBins * 4) + round256((uint64_t)s.tiles * 2 * cols * 4);
}

int elx_embedding_bwd(const void *index, int index_bytes, uint64_t n, const void *dy, uint64_t dy_stride, void *dtable, uint64_t vocab,
                      uint32_t cols, float scale, int64_t padding, void *workspace, uint64_t workspace_bytes, int dtype, void *stream) {
    if (!index || !dy || !dtable || !workspace) return ELX_E_NULL;
    if (!is_float_code(dtype) || (index_bytes != 4 && index_bytes != 8)) return ELX_E_DTYPE;
    if (n == 0 || n > kMaxTokens || vocab == 0 || vocab > kMaxVocab || cols == 0 || cols > kMaxCols) return ELX_E_SIZE;
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
    uint32_t *counts = (uint32_t *)at;
    at += round256((uint64_t)s.sort_blocks * kMaxBins * 4);
    float *partials = (float *)at;

    // dW is cleared in equal parts by the launches of the sort
    const uint64_t table_bytes = vocab * cols * es;
    const uint32_t parts = 2u * s.passes;
    const uint64_t per_part = (table_bytes / parts + kFillBytes) / kFillBytes * kFillBytes;
    uint32_t part = 0;
    hipStream_t st = (hipStream_t)stream;
    auto next_fill = [&](uint32_t &blocks) {
        const uint64_t begin = per_part * part < table_bytes ? per_part * part : table_bytes;
        ++part;
        const uint64_t end = part == parts || begin + per_part > table_bytes ? table_bytes : begin + per_part;
        blocks = (uint32_t)((end - begin + kFillBytes - 1) / kFillBytes);
        return Fill{(char *)dtable + begin, end - begin, aligned16(dtable) ? 16u : es};
    };
    for (int pass = 0; pass < s.passes; ++pass) {
        const Keys in = {index, index_bytes == 8, pass ? keys[(pass - 1) & 1] : nullptr, pass ? positions[(pass - 1) & 1] : nullptr, vocab,
                         padding};
        uint32_t blocks;
        Fill f = next_fill(blocks);
        hipLaunchKernelGGL(count_kernel, dim3(s.sort_blocks + blocks), dim3(kSortThreads), 0, st, in, n, s.per_block, s.sort_blocks,
                           pass * s.bits, 1u << s.bits, counts, f);
        if (int rc = (int)hipGetLastError()) return rc;
        f = next_fill(blocks);
        hipLaunchKernelGGL(scatter_kernel, dim3(s.sort_blocks + blocks), dim3(kSortThreads), 0, st, in, n, s.per_block, s.sort_blocks,
                           pass * s.bits, s.bits, counts, keys[pass & 1], positions[pass & 1], f);
        if (int rc = (int)hipGetLastError()) return rc;
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
