// Layer norm over the last dimension, forward and backward (include/elx_ops.h).
//
//   y = (x - mean) * rstd * w + b,  mean and var over a row, rstd = 1 / sqrt(var + eps)
//   with h = (x - mean) * rstd and t = dy * w:
//   dx = rstd * (t - mean(t) - h * mean(t * h)),   dw = sum over rows of dy * h,   db = sum over rows of dy
//
// A row is held in registers from its one read to its one write: W wavefronts per row, N accesses of V elements per lane.
// Short rows (a norm over the heads of attention) share a wavefront: L lanes per row, 64 / L rows (262144 x 64 bf16: 13 us
// forward and 23 us backward, against 62 and 93 with a wavefront per row).
// The variance is taken from the centred values in a second pass over the registers, so a large mean costs no digits.  All
// sums are in fp32 (per lane, then inside the wavefront, then over wavefronts through LDS), the one rounding to the
// tensor's type is at the store.
//
// Backward of few rows: one launch, some workgroups for dx, some for dw and db (layer_norm_few_kernel).  Of many: a workgroup of
// 16 wavefronts has 16 / W rows in flight and walks over rows with a stride; each lane sums dw and
// db of its own columns in registers over all its rows.  The row groups of a workgroup are added up in LDS, one partial row
// per workgroup goes to a workspace, and a second launch adds the partial rows up in a fixed order: no atomics, the same
// result every time.
//
// Both passes are bound by HBM where rows are many: 16384 x 4096 fp32 takes 93 us forward and 116 us backward from memory
// (0.54 and 0.81 GB: 5.8 and 6.9 TB/s; 77 us forward where the cache holds a part), 8192 x 2048 bf16 12.3 and 19.6 us, where
// the start and the end of a launch show.  A single row takes 2 us forward.  dw and db of many rows
// cost a second launch of 4 to 5 us; 512 x 2048 bf16 takes 3.7 and 5.1 us.
#include "elx_ops_device.h"

using namespace elx_ops;

namespace {

template <int D, int V>
struct Pack;    // V elements of type D as one access
template <>
struct Pack<ELX_F32, 4> {
    typedef f32x4 type;
};
template <>
struct Pack<ELX_F32, 1> {
    typedef float type;
};
template <>
struct Pack<ELX_F16, 8> {
    typedef u16x8 type;
};
template <>
struct Pack<ELX_F16, 1> {
    typedef uint16_t type;
};
template <>
struct Pack<ELX_BF16, 8> {
    typedef u16x8 type;
};
template <>
struct Pack<ELX_BF16, 1> {
    typedef uint16_t type;
};

template <int D, int V>
__device__ __forceinline__ void unpack(const typename Pack<D, V>::type &p, float (&x)[V]) {
    if constexpr (V == 1) {
        x[0] = Elem<D>::to_f32(p);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] = Elem<D>::to_f32(p[k]);
    }
}
template <int D, int V>
__device__ __forceinline__ typename Pack<D, V>::type pack(const float (&x)[V]) {
    typename Pack<D, V>::type p;
    if constexpr (V == 1) {
        p = Elem<D>::from_f32(x[0]);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) p[k] = Elem<D>::from_f32(x[k]);
    }
    return p;
}

template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_add(float x) {
    const int y = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xF, false);
    return x + __builtin_bit_cast(float, y);
}
// sum over L neighbouring lanes, the same in each of them
template <int L>
__device__ __forceinline__ float lanes_sum(float x) {
    if constexpr (L >= 2) x = dpp_add<0xB1, 0xF>(x);     // lanes 1 0 3 2 of each quad
    if constexpr (L >= 4) x = dpp_add<0x4E, 0xF>(x);     // lanes 2 3 0 1
    if constexpr (L >= 8) x = dpp_add<0x141, 0xF>(x);    // mirrored within 8
    if constexpr (L >= 16) x = dpp_add<0x140, 0xF>(x);   // mirrored within 16
    if constexpr (L == 32)                               // lanes 16 apart
        x += __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, x), 0x401F));
    if constexpr (L == 64) {
        x = dpp_add<0x142, 0xA>(x);
        x = dpp_add<0x143, 0xC>(x);
        x = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
    }
    return x;
}

// Sum over the W wavefronts of a row; `part` is W floats of LDS that belong to this row and this sum.  Every thread of the
// workgroup calls it.
template <int W, int L>
__device__ __forceinline__ float row_sum(float x, float *part, int wave) {
    static_assert(W == 1 || L == kWave, "rows that share a wavefront lie in it");
    x = lanes_sum<L>(x);
    if constexpr (W == 1) return x;
    if (threadIdx.x % kWave == 0) part[wave] = x;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) s += part[i];
    return s;
}

// ---------------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------------

// Workgroups of max(4, W) wavefronts; with W == 1 each has 64 / L rows of its own.
template <int D, int V, int N, int W, int L>
__global__ __launch_bounds__(kWave *(W > 4 ? W : 4)) void layer_norm_fwd_kernel(
    const typename Elem<D>::scalar *__restrict__ x, const typename Elem<D>::scalar *__restrict__ w,
    const typename Elem<D>::scalar *__restrict__ b, typename Elem<D>::scalar *__restrict__ y, float *__restrict__ mean_out,
    float *__restrict__ rstd_out, uint64_t rows, uint32_t cols, uint64_t x_stride, float eps) {
    typedef typename Pack<D, V>::type pack_t;
    constexpr int kGroups = (W > 4 ? 1 : 4 / W) * (kWave / L);    // rows of a workgroup
    __shared__ float part[2][kGroups][W];
    const int wave = threadIdx.x / kWave % W, lane = threadIdx.x % L;
    const int group = threadIdx.x / kWave / W * (kWave / L) + threadIdx.x % kWave / L;
    const uint64_t row = (uint64_t)blockIdx.x * kGroups + group;
    const bool live = row < rows;
    float v[N][V];
    float s = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const uint32_t c = ((uint32_t)(n * W + wave) * L + lane) * V;
#pragma unroll
        for (int k = 0; k < V; ++k) v[n][k] = 0.0f;
        if (live && c < cols) unpack<D, V>(*reinterpret_cast<const pack_t *>(x + row * x_stride + c), v[n]);
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int k = 0; k < V; ++k) s += v[n][k];
    const float inv = 1.0f / (float)cols;
    const float mean = row_sum<W, L>(s, part[0][group], wave) * inv;
    float q = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const uint32_t c = ((uint32_t)(n * W + wave) * L + lane) * V;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            v[n][k] -= mean;
            if (c < cols) q = fmaf(v[n][k], v[n][k], q);
        }
    }
    const float rstd = 1.0f / sqrtf(row_sum<W, L>(q, part[1][group], wave) * inv + eps);
    if (!live) return;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const uint32_t c = ((uint32_t)(n * W + wave) * L + lane) * V;
        if (c < cols) {
            float o[V], t[V];
#pragma unroll
            for (int k = 0; k < V; ++k) o[k] = v[n][k] * rstd;
            if (w) {
                unpack<D, V>(*reinterpret_cast<const pack_t *>(w + c), t);
#pragma unroll
                for (int k = 0; k < V; ++k) o[k] *= t[k];
            }
            if (b) {
                unpack<D, V>(*reinterpret_cast<const pack_t *>(b + c), t);
#pragma unroll
                for (int k = 0; k < V; ++k) o[k] += t[k];
            }
            __builtin_nontemporal_store(pack<D, V>(o), reinterpret_cast<pack_t *>(y + row * cols + c));
        }
    }
    if (wave == 0 && lane == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
}

// ---------------------------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------------------------

// The compiler may not reuse what it has computed from `x` before.
template <typename T>
__device__ __forceinline__ void forget(T &x) {
    if constexpr (sizeof(T) == 16) {
        u32x4 y = __builtin_bit_cast(u32x4, x);
        asm volatile("" : "+v"(y));
        x = __builtin_bit_cast(T, y);
    } else {    // one element
        asm volatile("" : "+v"(x));
    }
}

// One element of a row as a buffer of its own, at a byte offset: behind its end a load gives zero and a store does nothing.
template <int D>
__device__ __forceinline__ typename Elem<D>::scalar row_load(__amdgpu_buffer_rsrc_t r, uint32_t at) {
    if constexpr (D == ELX_F32)
        return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, (int)at, 0, 0));
    else
        return (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, (int)at, 0, 0);
}
template <int D>
__device__ __forceinline__ void row_store(__amdgpu_buffer_rsrc_t r, uint32_t at, typename Elem<D>::scalar x) {
    if constexpr (D == ELX_F32)
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, x), r, (int)at, 0, 2);    // non-temporal
    else
        __builtin_amdgcn_raw_buffer_store_b16(x, r, (int)at, 0, 2);
}

constexpr int kBwdWaves = 16;
constexpr int kBwdThreads = kBwdWaves * kWave;
constexpr uint32_t kBwdBlocks = 256;    // one workgroup per compute unit
// x and dy that fit the memory-side cache are likely to be there, left by the launches before: ordinary loads (8192 x 4096
// bf16: 41 us against 47 with non-temporal ones); what does not streams past it (16384 x 4096 fp32: 135 us against 144)
constexpr uint64_t kCacheBytes = 256ull << 20;

template <int D, int V, int N, int W, int L, bool STREAM>
__global__ __launch_bounds__(kBwdThreads) void layer_norm_bwd_kernel(
    const typename Elem<D>::scalar *__restrict__ dy, const typename Elem<D>::scalar *__restrict__ x,
    const typename Elem<D>::scalar *__restrict__ w, const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
    typename Elem<D>::scalar *__restrict__ dx, float *__restrict__ partials, uint64_t rows, uint32_t cols, uint64_t dy_stride,
    uint64_t x_stride) {
    typedef typename Pack<D, V>::type pack_t;
    constexpr int kGroups = kBwdWaves / W * (kWave / L);    // rows in flight
    constexpr bool kAhead = V * N <= 8;    // a lane has 128 registers: no room for a second row beyond that
    // 16 elements one by one: with a 64-bit address and a mask for each access, and w held, registers spilled to memory (2000 x
    // 16383 fp32 695 us, bf16 127; 91 and 56 without).  The row is a buffer and an access one offset into it; the workgroup has one
    // row, so the buffer is the same in all lanes.
    constexpr bool kBuffer = V == 1 && N > 8;
    static_assert(!kBuffer || W == kBwdWaves, "a row per workgroup");
    // h and t are computed once more for dx where the registers to keep them are short; 8 elements of 16 wavefronts keep them
    // (8191 x 4097 bf16 107 us, 111 with them computed again; 2047 x 769 fp16, two wavefronts, 8.0 and 6.8).
    constexpr bool kOnceMore = V > 1 || kBuffer || W < kBwdWaves;
    const uint32_t row_bytes = cols * (uint32_t)sizeof(typename Elem<D>::scalar);
    constexpr int kUnrollSums = kBuffer ? 4 : W;
    __shared__ float part[2][2][W > 1 ? kGroups : 1][W];
    const int wave = threadIdx.x / kWave % W, lane = threadIdx.x % L;
    const int group = W == kBwdWaves ? 0 : threadIdx.x / kWave / W * (kWave / L) + threadIdx.x % kWave / L;
    const uint32_t first = ((uint32_t)wave * L + lane) * (uint32_t)sizeof(pack_t);    // byte offset of this lane's first access
    auto offset_of = [&](int n) { return first + (uint32_t)n * (W * L * (uint32_t)sizeof(pack_t)); };
    float dw[N][V], db[N][V];
    pack_t pw[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const uint32_t c = ((uint32_t)(n * W + wave) * L + lane) * V;
        float one[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            dw[n][k] = db[n][k] = 0.0f;
            one[k] = 1.0f;
        }
        if constexpr (!kBuffer) pw[n] = w && c < cols ? *reinterpret_cast<const pack_t *>(w + c) : pack<D, V>(one);
    }
    const float inv = 1.0f / (float)cols;
    // every wavefront takes the same number of turns: the barriers inside are the workgroup's
    const uint64_t per_turn = (uint64_t)gridDim.x * kGroups;
    const uint64_t turns = (rows + per_turn - 1) / per_turn;
    pack_t px[N], pg[N];
    float mean, rstd;
    auto fetch = [&](uint64_t turn, pack_t (&qx)[N], pack_t (&qg)[N], float &m, float &r) {
        const uint64_t row = turn * per_turn + (uint64_t)blockIdx.x * kGroups + group;
        const bool live = row < rows;
        m = live ? mean_in[row] : 0.0f;
        r = live ? rstd_in[row] : 0.0f;
        const __amdgpu_buffer_rsrc_t rx = tile_rsrc(kBuffer && live ? x + row * x_stride : x, kBuffer && live ? row_bytes : 0);
        const __amdgpu_buffer_rsrc_t rg = tile_rsrc(kBuffer && live ? dy + row * dy_stride : dy, kBuffer && live ? row_bytes : 0);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const uint32_t c = ((uint32_t)(n * W + wave) * L + lane) * V;
            if constexpr (kBuffer) {
                qx[n] = row_load<D>(rx, offset_of(n));
                qg[n] = row_load<D>(rg, offset_of(n));
                continue;
            }
            qx[n] = pack_t{};
            qg[n] = pack_t{};
            if (live && c < cols) {
                const pack_t *at = reinterpret_cast<const pack_t *>(x + row * x_stride + c);
                const pack_t *from = reinterpret_cast<const pack_t *>(dy + row * dy_stride + c);
                if constexpr (STREAM) {
                    qx[n] = __builtin_nontemporal_load(at);
                    qg[n] = __builtin_nontemporal_load(from);
                } else {
                    qx[n] = *at;
                    qg[n] = *from;
                }
            }
        }
    };
    const __amdgpu_buffer_rsrc_t rw = tile_rsrc(kBuffer && w ? w : x, kBuffer && w ? row_bytes : 0);
    auto weight_of = [&](int n, float (&wt)[V]) {
        if constexpr (kBuffer) {    // from the cache, twice: there is no room for it either
            const float got = Elem<D>::to_f32(row_load<D>(rw, offset_of(n)));
            wt[0] = w ? got : 1.0f;
        } else {
            unpack<D, V>(pw[n], wt);
        }
    };
    fetch(0, px, pg, mean, rstd);
    pack_t nx[N], ng[N];
    float next_mean = 0.0f, next_rstd = 0.0f;
    if constexpr (kAhead) {
        if (turns > 1) fetch(1, nx, ng, next_mean, next_rstd);
    }
    for (uint64_t turn = 0; turn < turns; ++turn) {
        const uint64_t row = turn * per_turn + (uint64_t)blockIdx.x * kGroups + group;
        // the next two rows are on their way while this one is summed, waits at the barrier and is written
        pack_t lx[N], lg[N];
        float later_mean = 0.0f, later_rstd = 0.0f;
        if constexpr (kAhead) {
            if (turn + 2 < turns) fetch(turn + 2, lx, lg, later_mean, later_rstd);
        }
        float st = 0.0f, sth = 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const uint32_t c = ((uint32_t)(n * W + wave) * L + lane) * V;
            float h[V], g[V], wt[V];
            unpack<D, V>(px[n], h);
            unpack<D, V>(pg[n], g);
            weight_of(n, wt);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                h[k] = kBuffer || c < cols ? (h[k] - mean) * rstd : 0.0f;
                dw[n][k] = fmaf(g[k], h[k], dw[n][k]);
                db[n][k] += g[k];
                const float t = g[k] * wt[k];
                st += t;
                sth = fmaf(t, h[k], sth);
            }
        }
        // two sums share a barrier; the buffers alternate, so a wavefront that is a turn ahead writes elsewhere
        st = lanes_sum<L>(st);
        sth = lanes_sum<L>(sth);
        if constexpr (W > 1) {
            float *p = part[turn & 1][0][group], *q = part[turn & 1][1][group];
            if (lane == 0) {
                p[wave] = st;
                q[wave] = sth;
            }
            __syncthreads();
            st = sth = 0.0f;
#pragma unroll kUnrollSums
            for (int i = 0; i < W; ++i) {
                st += p[i];
                sth += q[i];
            }
        }
        st *= inv;
        sth *= inv;
        if (row < rows && dx) {    // h and t once more, from the row as it came: cheaper than the registers to keep them
            const __amdgpu_buffer_rsrc_t rd = tile_rsrc(kBuffer ? dx + row * cols : dx, kBuffer ? row_bytes : 0);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                if constexpr (kOnceMore) {
                    forget(px[n]);
                    forget(pg[n]);
                    if constexpr (!kBuffer) forget(pw[n]);
                }
                const uint32_t c = ((uint32_t)(n * W + wave) * L + lane) * V;
                if (kBuffer || c < cols) {
                    float h[V], g[V], wt[V], o[V];
                    unpack<D, V>(px[n], h);
                    unpack<D, V>(pg[n], g);
                    weight_of(n, wt);
#pragma unroll
                    for (int k = 0; k < V; ++k) o[k] = (g[k] * wt[k] - st - (h[k] - mean) * rstd * sth) * rstd;
                    if constexpr (kBuffer)
                        row_store<D>(rd, offset_of(n), pack<D, V>(o));
                    else
                        __builtin_nontemporal_store(pack<D, V>(o), reinterpret_cast<pack_t *>(dx + row * cols + c));
                }
            }
        }
        if constexpr (kAhead) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                px[n] = nx[n];
                pg[n] = ng[n];
                nx[n] = lx[n];
                ng[n] = lg[n];
            }
            mean = next_mean;
            rstd = next_rstd;
            next_mean = later_mean;
            next_rstd = later_rstd;
        } else if (turn + 1 < turns) {
            fetch(turn + 1, px, pg, mean, rstd);
        }
    }
    if (!partials) return;
    // rows that share a wavefront first
#pragma unroll
    for (int d = L; d < kWave; d <<= 1)
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                dw[n][k] += __shfl_xor(dw[n][k], d, kWave);
                db[n][k] += __shfl_xor(db[n][k], d, kWave);
            }
    // add the groups of wavefronts up, dw then db, through one buffer of LDS
    constexpr int kSums = kBwdWaves / W;
    __shared__ float sums[kSums > 1 ? kSums * W * L * V * N : 1];
    constexpr uint32_t kWidth = W * L * V * N;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float *out = partials + ((uint64_t)blockIdx.x * 2 + which) * cols;
        if constexpr (kSums > 1) {
            __syncthreads();
            if (threadIdx.x % kWave < L) {
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int k = 0; k < V; ++k)
                        sums[threadIdx.x / kWave / W * kWidth + ((uint32_t)(n * W + wave) * L + lane) * V + k] = which ? db[n][k] : dw[n][k];
            }
            __syncthreads();
            for (uint32_t c = threadIdx.x; c < cols; c += kBwdThreads) {
                float s = 0.0f;
#pragma unroll
                for (int g = 0; g < kSums; ++g) s += sums[g * kWidth + c];
                out[c] = s;
            }
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const uint32_t c = ((uint32_t)(n * W + wave) * L + lane) * V + k;
                    if (c < cols) out[c] = which ? db[n][k] : dw[n][k];
                }
        }
    }
}

// Adds the partial rows up: 64 columns of dw or db per workgroup, its 16 wavefronts take every 16th partial row.
template <int D>
__global__ __launch_bounds__(kBwdThreads) void layer_norm_fold_kernel(const float *__restrict__ partials, uint32_t blocks,
                                                                      uint32_t cols, typename Elem<D>::scalar *dw,
                                                                      typename Elem<D>::scalar *db) {
    __shared__ float sums[kBwdWaves][kWave];
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const uint32_t c = blockIdx.x * kWave + lane, which = blockIdx.y;
    float x[kBwdBlocks / kBwdWaves];    // all on their way at once
#pragma unroll
    for (uint32_t i = 0; i < kBwdBlocks / kBwdWaves; ++i) {
        const uint32_t r = i * kBwdWaves + wave;
        x[i] = c < cols && r < blocks ? partials[((uint64_t)r * 2 + which) * cols + c] : 0.0f;
    }
    float s = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kBwdBlocks / kBwdWaves; ++i) s += x[i];
    sums[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < cols) {
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < kBwdWaves; ++i) s += sums[i][lane];
        typename Elem<D>::scalar *out = which ? db : dw;
        if (out) out[c] = Elem<D>::from_f32(s);
    }
}

// Few rows: dx and the sums over rows side by side in one launch; mean and rstd are there, so neither needs the other.  The
// first `chunks` workgroups take `col_lanes` * V columns of dw and db each, over all rows; those behind them rows of dx.
constexpr int kFewThreads = 4 * kWave;

template <int D, int V, int N, int W, int L>
__global__ __launch_bounds__(kFewThreads) void layer_norm_few_kernel(
    const typename Elem<D>::scalar *__restrict__ dy, const typename Elem<D>::scalar *__restrict__ x,
    const typename Elem<D>::scalar *__restrict__ w, const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
    typename Elem<D>::scalar *__restrict__ dx, typename Elem<D>::scalar *__restrict__ dw, typename Elem<D>::scalar *__restrict__ db,
    uint32_t rows, uint32_t cols, uint64_t dy_stride, uint64_t x_stride, uint32_t chunks, uint32_t col_lanes) {
    typedef typename Pack<D, V>::type pack_t;
    static_assert(W <= 4, "a workgroup has four wavefronts");
    if (blockIdx.x < chunks) {
        constexpr uint32_t kAhead = 4;
        __shared__ float sums[2][kFewThreads * V];
        const uint32_t groups = kFewThreads / col_lanes, width = col_lanes * V;
        const uint32_t group = threadIdx.x / col_lanes, c0 = blockIdx.x * width, c = c0 + threadIdx.x % col_lanes * V;
        float sw[V], sb[V];
#pragma unroll
        for (int k = 0; k < V; ++k) sw[k] = sb[k] = 0.0f;
        for (uint32_t r0 = group; r0 < rows; r0 += groups * kAhead) {
            pack_t px[kAhead], pg[kAhead];
            float mean[kAhead], rstd[kAhead];
#pragma unroll
            for (uint32_t j = 0; j < kAhead; ++j) {    // on their way at once
                const uint32_t row = r0 + j * groups;
                px[j] = pg[j] = pack_t{};
                mean[j] = rstd[j] = 0.0f;
                if (row < rows && c < cols) {
                    px[j] = *reinterpret_cast<const pack_t *>(x + row * x_stride + c);
                    pg[j] = *reinterpret_cast<const pack_t *>(dy + row * dy_stride + c);
                    mean[j] = mean_in[row];
                    rstd[j] = rstd_in[row];
                }
            }
#pragma unroll
            for (uint32_t j = 0; j < kAhead; ++j) {
                float h[V], g[V];
                unpack<D, V>(px[j], h);
                unpack<D, V>(pg[j], g);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    sw[k] = fmaf(g[k], (h[k] - mean[j]) * rstd[j], sw[k]);
                    sb[k] += g[k];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < V; ++k) {
            sums[0][threadIdx.x * V + k] = sw[k];
            sums[1][threadIdx.x * V + k] = sb[k];
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < 2 * width; i += kFewThreads) {
            const uint32_t which = i / width, at = i % width;
            float s = 0.0f;
#pragma unroll 16
            for (uint32_t g = 0; g < groups; ++g) s += sums[which][g * width + at];
            typename Elem<D>::scalar *out = which ? db : dw;
            if (out && c0 + at < cols) out[c0 + at] = Elem<D>::from_f32(s);
        }
        return;
    }
    constexpr int kGroups = 4 / W * (kWave / L);    // rows of a workgroup
    __shared__ float part[2][kGroups][W];
    const int wave = threadIdx.x / kWave % W, lane = threadIdx.x % L;
    const int group = threadIdx.x / kWave / W * (kWave / L) + threadIdx.x % kWave / L;
    const uint32_t row = (blockIdx.x - chunks) * kGroups + group;
    const bool live = row < rows;
    const float mean = live ? mean_in[row] : 0.0f, rstd = live ? rstd_in[row] : 0.0f;
    float h[N][V], t[N][V], st = 0.0f, sth = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const uint32_t c = ((uint32_t)(n * W + wave) * L + lane) * V;
#pragma unroll
        for (int k = 0; k < V; ++k) h[n][k] = t[n][k] = 0.0f;
        if (live && c < cols) {
            unpack<D, V>(*reinterpret_cast<const pack_t *>(x + row * x_stride + c), h[n]);
            unpack<D, V>(*reinterpret_cast<const pack_t *>(dy + row * dy_stride + c), t[n]);
            if (w) {
                float wt[V];
                unpack<D, V>(*reinterpret_cast<const pack_t *>(w + c), wt);
#pragma unroll
                for (int k = 0; k < V; ++k) t[n][k] *= wt[k];
            }
#pragma unroll
            for (int k = 0; k < V; ++k) h[n][k] = (h[n][k] - mean) * rstd;
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int k = 0; k < V; ++k) {
            st += t[n][k];
            sth = fmaf(t[n][k], h[n][k], sth);
        }
    const float inv = 1.0f / (float)cols;
    st = row_sum<W, L>(st, part[0][group], wave) * inv;
    sth = row_sum<W, L>(sth, part[1][group], wave) * inv;
    if (!live) return;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const uint32_t c = ((uint32_t)(n * W + wave) * L + lane) * V;
        if (c < cols) {
            float o[V];
#pragma unroll
            for (int k = 0; k < V; ++k) o[k] = (t[n][k] - st - h[n][k] * sth) * rstd;
            __builtin_nontemporal_store(pack<D, V>(o), reinterpret_cast<pack_t *>(dx + (uint64_t)row * cols + c));
        }
    }
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------

constexpr uint32_t kMaxCols = 16384;
constexpr uint64_t kMaxRows = 1ull << 36, kMaxStride = 1ull << 36;
constexpr uint64_t kPieceRows = 1ull << 23;

struct Fwd {
    const void *x, *w, *b;
    void *y;
    float *mean, *rstd;
    uint64_t rows, x_stride;
    uint32_t cols;
    float eps;
    hipStream_t stream;
};

template <int D, int V, int N, int W, int L = kWave>
int launch_fwd(const Fwd &a) {
    typedef typename Elem<D>::scalar T;
    constexpr int groups = (W > 4 ? 1 : 4 / W) * (kWave / L);
    hipLaunchKernelGGL((layer_norm_fwd_kernel<D, V, N, W, L>), dim3((uint32_t)((a.rows + groups - 1) / groups)),
                       dim3(kWave * (W > 4 ? W : 4)), 0, a.stream, (const T *)a.x, (const T *)a.w, (const T *)a.b, (T *)a.y, a.mean,
                       a.rstd, a.rows, a.cols, a.x_stride, a.eps);
    return (int)hipGetLastError();
}

template <int N, int W, int L = kWave>
struct shape {    // accesses per lane, wavefronts per row, lanes per row of a wavefront
    static constexpr int accesses = N, waves = W, lanes = L;
};

// wavefronts per row and accesses per lane, the latter rounded up to what is compiled; FEW: fewer than 4096 rows
template <int V, bool FEW, typename F>
int dispatch_rows(uint64_t rows, uint32_t cols, F &&launch) {
    const uint32_t accesses = (cols + kWave * V - 1) / (kWave * V);    // wavefront-wide accesses of a row
    // Four wavefronts read a long row in a quarter of the steps, one wavefront needs no barrier:
    //   16384 x 4096 fp32   77 us with four, 93 with one      32768 x 2048 bf16   46 us with four, 42 with one
    //   32768 x 4096 bf16   79              100                8192 x 2048 bf16   14              10.6
    //    8191 x 1025 fp16   18               25                8191 x 1023 fp16   13.9            12.6
    // With few rows it is the steps that count (1024 x 2048 bf16: 4.5 us with four, 5.5 with one; 4096 x 2048: 7.1, 6.8).
    if (accesses >= (V == 1 ? 17 : 8) || ((FEW || rows < 4096) && accesses >= 4)) {
        const uint32_t n = (accesses + 3) / 4;
        if (n <= 1) return launch(shape<1, 4>());
        if (n <= 2) return launch(shape<2, 4>());
        if (n <= 4) return launch(shape<4, 4>());
        if (n <= 8) return launch(shape<8, 4>());
        if constexpr (V <= 4)
            if (n <= 16) return launch(shape<16, 4>());
        if constexpr (V == 1) {
            if (n <= 32) return launch(shape<32, 4>());
            if (n <= 64) return launch(shape<64, 4>());
        }
        return ELX_E_SIZE;
    }
    if (cols <= 4 * V) return launch(shape<1, 1, 4>());
    if (cols <= 8 * V) return launch(shape<1, 1, 8>());
    if (cols <= 16 * V) return launch(shape<1, 1, 16>());
    if (cols <= 32 * V) return launch(shape<1, 1, 32>());
    if (accesses <= 1) return launch(shape<1, 1>());
    if (accesses <= 2) return launch(shape<2, 1>());
    if (accesses <= 4) return launch(shape<4, 1>());
    if constexpr (!FEW) {
        if (accesses <= 8) return launch(shape<8, 1>());
        if constexpr (V == 1)
            if (accesses <= 16) return launch(shape<16, 1>());
    }
    return ELX_E_SIZE;
}

template <int D, int V>
int dispatch_fwd(const Fwd &a) {
    return dispatch_rows<V, false>(a.rows, a.cols, [&](auto s) { return launch_fwd<D, V, s.accesses, s.waves, s.lanes>(a); });
}

struct Bwd {
    const void *dy, *x, *w;
    const float *mean, *rstd;
    void *dx, *dw, *db;
    float *partials;
    uint64_t rows, dy_stride, x_stride;
    uint32_t cols;
    hipStream_t stream;
};

// Wavefronts per row of the backward pass: 8 elements per lane.  With 16 there is no room for the next rows (8192 x 4096 bf16:
// 42 us against 38); with 4 of one element each, more wavefronts wait for each other (8191 x 2049 fp16: 58 against 49).
uint32_t bwd_waves(uint32_t cols) {
    uint32_t w = 1;
    while (w < 16 && w * kWave * 8 < cols) w *= 2;
    return w;
}

template <int D, int V, int N, int W, int L = kWave>
int launch_bwd(const Bwd &a) {
    typedef typename Elem<D>::scalar T;
    constexpr uint32_t groups = kBwdWaves / W * (kWave / L);
    const uint64_t want = (a.rows + groups - 1) / groups;
    const uint32_t blocks = (uint32_t)(want < kBwdBlocks ? want : kBwdBlocks);
    auto kernel = layer_norm_bwd_kernel<D, V, N, W, L, false>;
    if constexpr (V > 1) {
        if (2 * a.rows * a.cols * sizeof(T) > kCacheBytes) kernel = layer_norm_bwd_kernel<D, V, N, W, L, true>;
    }
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kBwdThreads), 0, a.stream, (const T *)a.dy, (const T *)a.x, (const T *)a.w, a.mean,
                       a.rstd, (T *)a.dx, a.partials, a.rows, a.cols, a.dy_stride, a.x_stride);
    if (int rc = (int)hipGetLastError()) return rc;
    if (!a.partials) return 0;
    hipLaunchKernelGGL((layer_norm_fold_kernel<D>), dim3((a.cols + kWave - 1) / kWave, 2), dim3(kBwdThreads), 0, a.stream, a.partials,
                       blocks, a.cols, (T *)a.dw, (T *)a.db);
    return (int)hipGetLastError();
}

// Up to that many rows go in one launch (512 x 2048 bf16: 5.1 us against 9.8 in two, 1024 rows 6.9 against 10.9; 1400 rows of
// 4096 17 against 15.7), with 64 or 128 bytes of a row per workgroup of the sums: the narrower, the more workgroups, the wider,
// the better the reads (1024 x 2048 bf16 6.9 us with 64 and 9.4 with 128, 1024 x 11008 bf16 26 and 20).
constexpr uint64_t kFewRows = 1024;
static_assert(kFewRows < 4096, "FEW of dispatch_rows");
constexpr uint32_t kNarrowBytes = 6144;    // of a row

template <int D, int V, int N, int W, int L>
int launch_few(const Bwd &a) {
    typedef typename Elem<D>::scalar T;
    constexpr uint32_t groups = 4 / W * (kWave / L);
    const uint32_t col_lanes = a.cols * sizeof(T) <= kNarrowBytes ? 4 : 8;
    const uint32_t width = col_lanes * V, rows = (uint32_t)a.rows;
    const uint32_t chunks = a.dw || a.db ? (a.cols + width - 1) / width : 0;
    hipLaunchKernelGGL((layer_norm_few_kernel<D, V, N, W, L>), dim3(chunks + (a.dx ? (rows + groups - 1) / groups : 0)), dim3(kFewThreads), 0,
                       a.stream, (const T *)a.dy, (const T *)a.x, (const T *)a.w, a.mean, a.rstd, (T *)a.dx, (T *)a.dw, (T *)a.db, rows,
                       a.cols, a.dy_stride, a.x_stride, chunks, col_lanes);
    return (int)hipGetLastError();
}


template <int D, int V>
int dispatch_bwd(const Bwd &a) {
    if (a.rows <= kFewRows)
        return dispatch_rows<V, true>(a.rows, a.cols, [&](auto s) { return launch_few<D, V, s.accesses, s.waves, s.lanes>(a); });
    if (a.cols <= 4 * V) return launch_bwd<D, V, 1, 1, 4>(a);
    if (a.cols <= 8 * V) return launch_bwd<D, V, 1, 1, 8>(a);
    if (a.cols <= 16 * V) return launch_bwd<D, V, 1, 1, 16>(a);
    if (a.cols <= 32 * V) return launch_bwd<D, V, 1, 1, 32>(a);
    const uint32_t waves = bwd_waves(a.cols);
    const uint32_t n = (a.cols + waves * kWave * V - 1) / (waves * kWave * V);
    // more than one wavefront: cols > 256 waves, which is more than 4 elements per lane
#define ELX_CASE(WAVES, ACCESSES)                                                  \
    if constexpr (ACCESSES * V <= (WAVES == 16 ? 16 : 8) && (WAVES == 1 || ACCESSES * V > 4)) \
        if (waves == WAVES && n <= ACCESSES) return launch_bwd<D, V, ACCESSES, WAVES>(a);
    ELX_CASE(1, 1)
    ELX_CASE(1, 2)
    ELX_CASE(1, 4)
    ELX_CASE(1, 8)
    ELX_CASE(2, 1)
    ELX_CASE(2, 2)
    ELX_CASE(2, 4)
    ELX_CASE(2, 8)
    ELX_CASE(4, 1)
    ELX_CASE(4, 2)
    ELX_CASE(4, 4)
    ELX_CASE(4, 8)
    ELX_CASE(8, 1)
    ELX_CASE(8, 2)
    ELX_CASE(8, 4)
    ELX_CASE(8, 8)
    ELX_CASE(16, 1)
    ELX_CASE(16, 2)
    ELX_CASE(16, 4)
    ELX_CASE(16, 8)
    ELX_CASE(16, 16)
#undef ELX_CASE
    return ELX_E_SIZE;
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

}    // namespace

extern "C" {

uint32_t elx_layer_norm_max_cols(void) { return kMaxCols; }

uint64_t elx_layer_norm_bwd_workspace(uint64_t rows, uint32_t cols) {
    const uint64_t most = rows < kBwdBlocks ? rows : kBwdBlocks;
    return most * 2 * cols * sizeof(float);
}

int elx_layer_norm_fwd(const void *x, const void *w, const void *b, void *y, float *mean, float *rstd, uint64_t rows, uint32_t cols,
                       uint64_t x_stride, float eps, int dtype, void *stream) {
    if (!x || !y) return ELX_E_NULL;
    if (!is_float_code(dtype)) return ELX_E_DTYPE;
    if (rows == 0 || rows > kMaxRows || cols == 0 || cols > kMaxCols) return ELX_E_SIZE;
    if ((x_stride < cols && rows > 1) || x_stride > kMaxStride) return ELX_E_RANGE;
    const uint32_t es = elem_size(dtype), v = 16 / es;
    if ((((uintptr_t)x | (uintptr_t)y | (uintptr_t)w | (uintptr_t)b) & (es - 1)) || (((uintptr_t)mean | (uintptr_t)rstd) & 3u))
        return ELX_E_ALIGN;
    const bool vec = aligned16(x) && aligned16(y) && aligned16(w) && aligned16(b) && cols % v == 0 && x_stride % v == 0;
    // a launch has at most 2^32 threads: rows in pieces
    for (uint64_t r = 0; r < rows; r += kPieceRows) {
        const Fwd a = {(const char *)x + r * x_stride * es, w, b, (char *)y + r * cols * es, mean ? mean + r : nullptr,
                       rstd ? rstd + r : nullptr, rows - r < kPieceRows ? rows - r : kPieceRows, x_stride, cols, eps,
                       (hipStream_t)stream};
        int rc;
        switch (dtype) {
            case ELX_F32: rc = vec ? dispatch_fwd<ELX_F32, 4>(a) : dispatch_fwd<ELX_F32, 1>(a); break;
            case ELX_F16: rc = vec ? dispatch_fwd<ELX_F16, 8>(a) : dispatch_fwd<ELX_F16, 1>(a); break;
            default: rc = vec ? dispatch_fwd<ELX_BF16, 8>(a) : dispatch_fwd<ELX_BF16, 1>(a);
        }
        if (rc) return rc;
    }
    return 0;
}

int elx_layer_norm_bwd(const void *dy, const void *x, const void *w, const float *mean, const float *rstd, void *dx, void *dw, void *db,
                       void *workspace, uint64_t workspace_bytes, uint64_t rows, uint32_t cols, uint64_t dy_stride, uint64_t x_stride,
                       int dtype, void *stream) {
    if (!dy || !x || !mean || !rstd || (!dx && !dw && !db)) return ELX_E_NULL;
    if (!is_float_code(dtype)) return ELX_E_DTYPE;
    if (rows == 0 || rows > kMaxRows || cols == 0 || cols > kMaxCols) return ELX_E_SIZE;
    if (((x_stride < cols || dy_stride < cols) && rows > 1) || x_stride > kMaxStride || dy_stride > kMaxStride) return ELX_E_RANGE;
    const bool sums = dw || db;
    if (sums && (!workspace || workspace_bytes < elx_layer_norm_bwd_workspace(rows, cols))) return !workspace ? ELX_E_NULL : ELX_E_SIZE;
    const uint32_t es = elem_size(dtype), v = 16 / es;
    if ((((uintptr_t)dy | (uintptr_t)x | (uintptr_t)w | (uintptr_t)dx | (uintptr_t)dw | (uintptr_t)db) & (es - 1)) ||
        (((uintptr_t)mean | (uintptr_t)rstd | (uintptr_t)workspace) & 3u))
        return ELX_E_ALIGN;
    const Bwd a = {dy, x, w, mean, rstd, dx, dw, db, sums ? (float *)workspace : nullptr, rows, dy_stride, x_stride, cols, (hipStream_t)stream};
    const bool vec = aligned16(dy) && aligned16(x) && aligned16(w) && aligned16(dx) && cols % v == 0 && x_stride % v == 0 && dy_stride % v == 0;
    switch (dtype) {
        case ELX_F32: return vec ? dispatch_bwd<ELX_F32, 4>(a) : dispatch_bwd<ELX_F32, 1>(a);
        case ELX_F16: return vec ? dispatch_bwd<ELX_F16, 8>(a) : dispatch_bwd<ELX_F16, 1>(a);
        default: return vec ? dispatch_bwd<ELX_BF16, 8>(a) : dispatch_bwd<ELX_BF16, 1>(a);
    }
}

}    // extern "C"
