// Adam / AdamW with exp_avg and exp_avg_sq held in 8 bits (include/elx_ops.h has the code).
//
//   adam8_step_kernel    unscale + Adam/AdamW on master and 8-bit moments + low-precision writeback
//   state8_read_kernel   codes -> fp32 / bf16 values
//   state8_write_kernel  fp32 values -> codes
//
// The step is one pass over its data: 16 bytes per element with 16-bit gradients (gradient 2, master 4 + 4, codes
// 2 + 2, low-precision copy 2) against the 28 of the 32-bit state.  A block of the code is the tile of one wavefront:
// 4 elements a lane, so that the largest magnitude of the block is a reduction inside one wavefront (four steps inside
// rows of 16 lanes, two between rows), and nothing goes through LDS.  The access pattern is that of the 32-bit update
// (elx_kernels.hip): one tile per workgroup, tiles in address order, the number of resident workgroups held by an LDS
// reservation that no thread touches.
//
// Bound by HBM: 1.31e9 elements (OPT-1.3B in bf16) take 3.17 to 3.19 ms = 6.6 TB/s, the rate of a copy, against 5.53 ms with the
// 32-bit state; 5.4e8 elements with fp32 gradients (20 bytes each) 1.69 ms = 6.4 TB/s against 2.57; 16 Mi fp32 elements whose data
// stay in the memory-side cache 39 us against 66.  Reading the values of 128 Mi elements takes 187 us to fp32 (7.2 TB/s) and 115 us
// to bf16 (7.0 TB/s) where the codes were read before, 134 us behind a step (6.0 TB/s).  Writing as many from fp32 takes 143 us a
// moment (4.7 TB/s): checkpoints are loaded with it, a step does not.
//
// Arithmetic: fp32; unscale and moments have the bits of the 32-bit update (fused multiply-adds written as fmaf,
// -ffp-contract=off), the change of the master weight is that update's to within 2^-20.  Only the new moments are rounded to
// 8 bits, after the master has used them.
#include "elx_ops_device.h"

#include "../elx_host.h"

using namespace elx_ops;

namespace {

using elx_host::kDivMulInv;
using elx_host::kDivNone;
using elx_host::kDivTrue;
using elx_host::Unscale;

constexpr uint32_t kTile = 256;
constexpr int kVec = 4;
static_assert(kTile == elx_host::kTile, "a tile of the update tables is a block of the 8-bit code");

// Resident workgroups per compute unit when the caller names no number.  1.3e9 elements in bf16: 3.40 ms with 16, 3.25 with 20,
// 3.29 with 24, 3.47 with 32; where the gradient is divided by a scale that is no power of two 3.30 with 20, 3.27 with 24: what is
// taken lies between.  5.4e8 elements in bf16: 1.31 ms with 18, 1.30 with 20, 22 and 24.
constexpr uint32_t kBlocksPerCu = 22;

// cache policy, as in the 32-bit update: everything streams; the low-precision copy stays in the memory-side cache; all does
enum { kStream = 0, kKeepLowp = 1, kKeepState = 2 };
template <int POLICY>
struct Aux {
    static constexpr int load = POLICY == kKeepState ? 0 : 2;
    static constexpr int store = POLICY == kKeepState ? 16 : 2 | 16;
    static constexpr int store_lowp = POLICY == kStream ? 2 | 16 : 16;
};

struct Hyper {
    float decay_mul, l2_wd, lerp_w, beta2, omb2, bc2_sqrt, eps, neg_step;
    uint32_t flags;
    float gate_div, gate_inv;
    uint32_t gate;
};

template <bool GATED>
__device__ __forceinline__ Hyper load_hyper(const ElxHyper *__restrict__ h) {
    Hyper r;
    r.gate_div = GATED ? h->gate_div_scale : -1.0f;
    r.gate_inv = GATED ? h->gate_inv_scale : 1.0f;
    r.gate = GATED ? h->gate : 0u;
    r.decay_mul = h->decay_mul;
    r.l2_wd = h->l2_wd;
    r.lerp_w = h->lerp_w;
    r.beta2 = h->beta2;
    r.omb2 = h->omb2;
    r.bc2_sqrt = h->bc2_sqrt;
    r.eps = h->eps;
    r.neg_step = h->neg_step;
    r.flags = h->flags;
    return r;
}

// sqrt and reciprocal instructions (1 ulp each) stand in for the IEEE sequences: with them a launch over 1.3 billion elements
// was bound by its vector work at any residency (3.47 ms at 32 workgroups per compute unit, 3.88 at 20), without them it is
// bound by HBM (3.25 ms at 20, and slower again beyond 24, like a copy).  Moments and codes do not depend on them; the change
// of a master weight is off by at most 2^-20 of itself.  The sqrt instruction takes subnormal numbers for zero: below this eps
// that would show, and the IEEE forms are taken.
constexpr float kFastEps = 0x1p-36f;

// One element, torch.optim.Adam's order of operations.  DIV: the gradient is divided by div_scale (else multiplied by
// inv_scale, which is exact, and 1 when nothing is unscaled); OPTIONS: L2 decay or the lerp from the gradient's end.
template <bool DIV, bool IEEE, bool OPTIONS>
__device__ __forceinline__ void adam_elem(float g, float &p, float &m, float &v, const Hyper &h, const Unscale &us, float rbc2) {
    g = DIV ? g / us.div_scale : g * us.inv_scale;
    p = p * h.decay_mul;
    if (OPTIONS && (h.flags & ELX_HYPER_L2)) g = fmaf(h.l2_wd, p, g);
    const float diff = g - m;
    m = fmaf(h.lerp_w, diff, OPTIONS && (h.flags & ELX_HYPER_LERP_FROM_G) ? g : m);
    v = fmaf(h.omb2 * g, g, v * h.beta2);
    if (IEEE) {
        p = p + (h.neg_step * m) / (sqrtf(v) / h.bc2_sqrt + h.eps);
    } else {
        const float denom = fmaf(__builtin_amdgcn_sqrtf(v), rbc2, h.eps);
        p = fmaf(h.neg_step * m, __builtin_amdgcn_rcpf(denom), p);
    }
}

// calls f with the variant of adam_elem that the launch-uniform choices select
template <typename F>
__device__ __forceinline__ void with_variant(const Hyper &h, const Unscale &us, F &&f) {
    const float rbc2 = __builtin_amdgcn_rcpf(h.bc2_sqrt);
    const uint32_t kind = (us.mode == kDivTrue ? 1u : 0u) | (h.eps >= kFastEps ? 0u : 2u) |
                          (h.flags & (ELX_HYPER_L2 | ELX_HYPER_LERP_FROM_G) ? 4u : 0u);
#define ELX_KIND(DIV, IEEE, OPTIONS)                                                                                          \
    case (DIV ? 1u : 0u) | (IEEE ? 2u : 0u) | (OPTIONS ? 4u : 0u):                                                            \
        f([&](float g, float &p, float &m, float &v) { adam_elem<DIV, IEEE, OPTIONS>(g, p, m, v, h, us, rbc2); });            \
        break;
    switch (kind) {
        ELX_KIND(false, false, false)
        ELX_KIND(true, false, false)
        ELX_KIND(false, true, false)
        ELX_KIND(true, true, false)
        ELX_KIND(false, false, true)
        ELX_KIND(true, false, true)
        ELX_KIND(false, true, true)
        default:
            f([&](float g, float &p, float &m, float &v) { adam_elem<true, true, true>(g, p, m, v, h, us, rbc2); });
    }
#undef ELX_KIND
}

// ---------------------------------------------------------------------------------------------
// the 8-bit code
// ---------------------------------------------------------------------------------------------

constexpr uint32_t kInf = 0x7F800000u;
// The largest magnitude that does not take exponent 255, 1.75 * 2^127.  Under 255 the code above these stands for 2^128, which
// fp32 does not hold: a finite value is held at 1.875 * 2^127 at most.
constexpr uint32_t kOrdinary = 0x7F600000u, kAvgTop = 0x77u, kSqTop = 0xF7u;
constexpr uint32_t kHalf = 1u << 19;    // r of rounding to nearest

__device__ __forceinline__ uint32_t mix(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x6A09E667u;
    x = (x ^ (x >> 15)) * 0xBB67AE85u;
    return x ^ (x >> 16);
}
constexpr uint32_t kGolden = 0x9E3779B9u;

__device__ __forceinline__ uint32_t block_key(uint32_t block, uint32_t salt, uint32_t step) {
    return mix(block ^ mix(salt * kGolden + step));
}
__device__ __forceinline__ uint32_t dither_of(uint32_t word, int k) {
    return __builtin_rotateright32(word, 8 * k) >> 12;
}

// Lanes without a partner get 0, the identity of max: the exchange then is an operand modifier of the max itself.
template <int CTRL, int ROWS>
__device__ __forceinline__ void dpp_max(uint32_t &x, uint32_t &y) {
    const uint32_t a = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, false);
    const uint32_t b = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)y, CTRL, ROWS, 0xF, false);
    x = x > a ? x : a;
    y = y > b ? y : b;
}
// Largest of the 64 lanes, in scalar registers, for two values at a time (each exchange has to wait two instructions for
// its operand: the other value's fill them).  Inside rows of 16 lanes: two exchanges inside quads, then of the halves of a
// row; then each row's last lane into the row behind it, then the lower half's into the upper.
__device__ __forceinline__ void wave_max(uint32_t &x, uint32_t &y) {
    dpp_max<0xB1, 0xF>(x, y);     // lanes 1 0 3 2 of each quad
    dpp_max<0x4E, 0xF>(x, y);     // lanes 2 3 0 1
    dpp_max<0x141, 0xF>(x, y);    // mirrored within 8 lanes
    dpp_max<0x140, 0xF>(x, y);    // mirrored within 16 lanes
    dpp_max<0x142, 0xA>(x, y);    // lane 15 of rows 0 and 2 into rows 1 and 3
    dpp_max<0x143, 0xC>(x, y);    // lane 31 into rows 2 and 3
    x = (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
    y = (uint32_t)__builtin_amdgcn_readlane((int)y, 63);
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }

// the exponent byte for a largest magnitude given by its bits: a fraction above 1.75 carries into the next exponent
__device__ __forceinline__ int exponent_of(uint32_t bits) { return (int)((bits + 0x1FFFFFu) >> 23); }

__device__ __forceinline__ void decode_avg(uint32_t word, int e, float (&m)[kVec]) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, true);
    m[0] = __builtin_ldexpf(lo[0], e - 135);
    m[1] = __builtin_ldexpf(lo[1], e - 135);
    m[2] = __builtin_ldexpf(hi[0], e - 135);
    m[3] = __builtin_ldexpf(hi[1], e - 135);
}

__device__ __forceinline__ void decode_sq(uint32_t word, int e, float (&v)[kVec]) {
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
        const uint32_t bits = (k < 3 ? word << (20 - 8 * k) : word >> 4) & 0x0FF00000u;
        v[k] = __builtin_ldexpf(__builtin_bit_cast(float, bits), e - 31);
    }
    // some byte is 255: the usual test for a zero byte, on the complement
    const uint32_t inv = ~word;
    if (__builtin_amdgcn_ballot_w64(((inv - 0x01010101u) & ~inv & 0x80808080u) != 0)) {
#pragma unroll
        for (int k = 0; k < kVec; ++k)
            if (((word >> (8 * k)) & 0xFFu) == 0xFFu) v[k] = __builtin_nanf("");
    }
}

// The moments of the wavefront's block -> four codes per lane and the two exponents.  Called by all 64 lanes.
__device__ __forceinline__ void encode(const float (&m)[kVec], const float (&v)[kVec], const uint32_t (&r)[kVec],
                                       uint32_t &m_word, uint32_t &v_word, int &me, int &ve) {
    uint32_t bm[kVec], bv[kVec];
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
        bm[k] = magnitude(m[k]);
        bv[k] = magnitude(v[k]);
    }
    uint32_t mt = max(max(bm[0], bm[1]), max(bm[2], bm[3])), vt = max(max(bv[0], bv[1]), max(bv[2], bv[3]));
    wave_max(mt, vt);
    const bool ordinary = max(mt, vt) <= kOrdinary;
    if (!ordinary) {    // the exponents are those of the finite elements
        mt = vt = 0;
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
            mt = max(mt, bm[k] < kInf ? bm[k] : 0u);
            vt = max(vt, bv[k] < kInf ? bv[k] : 0u);
        }
        wave_max(mt, vt);
    }
    me = exponent_of(mt);
    ve = exponent_of(vt);
    float x[kVec];
#pragma unroll
    for (int k = 0; k < kVec; ++k) x[k] = __builtin_ldexpf(m[k], 135 - me);
    int word = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    m_word = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], word, true);
    uint32_t code[kVec];
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
        // without its sign, which the code has no place for: a bit of it would land in the next element's code
        const uint32_t t = __builtin_bit_cast(uint32_t, __builtin_ldexpf(__builtin_fabsf(v[k]), 31 - ve));
        code[k] = max((t + r[k]) >> 20, min(bv[k], 1u));
    }
    if (!ordinary) {
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
            uint32_t c = (m_word >> (8 * k)) & 0xFFu;
            if (me == 255 && (c & 0x7Fu) > kAvgTop) c = (c & 0x80u) | kAvgTop;
            if (bm[k] >= kInf) c = 0x7Fu;
            m_word = (m_word & ~(0xFFu << (8 * k))) | (c << (8 * k));
            if (ve == 255) code[k] = min(code[k], kSqTop);
            if (bv[k] >= kInf) code[k] = 0xFFu;
        }
    }
    v_word = code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24;
}

// ---------------------------------------------------------------------------------------------
// the step
// ---------------------------------------------------------------------------------------------

struct Row {
    ElxChunk c;
    ElxState8 s;
};

// Both records of a row with one round trip of scalar loads.
__device__ __forceinline__ Row load_row(const ElxChunk *__restrict__ chunk, const ElxState8 *__restrict__ state) {
    const uint64_t *w = reinterpret_cast<const uint64_t *>(chunk);
    const uint64_t *u = reinterpret_cast<const uint64_t *>(state);
    uint64_t w0 = w[0], w1 = w[1], w2 = w[2], w3 = w[3], w4 = w[4], w5 = w[5], w6 = w[6], w8 = w[8], u0 = u[0], u1 = u[1];
    asm volatile("" : "+s"(w0), "+s"(w1), "+s"(w2), "+s"(w3), "+s"(w4), "+s"(w5), "+s"(w6), "+s"(w8), "+s"(u0), "+s"(u1));
    Row r;
    r.c.grad = reinterpret_cast<const void *>(w0);
    r.c.lowp_out = reinterpret_cast<void *>(w1);
    r.c.master = reinterpret_cast<float *>(w2);
    r.c.m = reinterpret_cast<float *>(w3);
    r.c.v = reinterpret_cast<float *>(w4);
    r.c.n_alloc = w5;
    r.c.n_valid = w6;
    r.c.tile_begin = 0;
    r.c.seg_begin = (uint32_t)w8;
    r.c.seg_end = (uint32_t)(w8 >> 32);
    r.s.scales = reinterpret_cast<uint16_t *>(u0);
    r.s.first_block = (uint32_t)u1;
    r.s.salt = (uint32_t)(u1 >> 32);
    return r;
}
static_assert(sizeof(ElxChunk) == 72 && sizeof(ElxState8) == 16, "load_row reads nine and two 64-bit words");

// Any tile, element by element: tiles that straddle a segment boundary, the partial tile at the end of a buffer, padding,
// buffers that are not 16-byte aligned.  The lanes hold the same elements as on the straight path, so that block and
// rounding are the same.  `s` is the first segment whose end is > base.
template <int GD, int LD, bool GATED>
__device__ __forceinline__ void tile_any(const Row &row, uint32_t tile, uint32_t tile_n, uint32_t s,
                                         const ElxSeg *__restrict__ segs, const ElxHyper *__restrict__ hypers,
                                         const Unscale &us_arg, bool refresh_only) {
    typedef typename Elem<GD>::scalar gscalar;
    const ElxChunk &c = row.c;
    const uint64_t base = (uint64_t)tile * kTile;
    const uint32_t lane = threadIdx.x;
    uint8_t *mc = reinterpret_cast<uint8_t *>(c.m) + base, *vc = reinterpret_cast<uint8_t *>(c.v) + base;
    float m[kVec], v[kVec];
    uint32_t r[kVec];
    bool changed = false;
    if (!refresh_only) {
        uint32_t mw = 0, vw = 0;
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
            const uint32_t i = lane * kVec + k;
            if (i < tile_n) {
                mw |= (uint32_t)mc[i] << (8 * k);
                vw |= (uint32_t)vc[i] << (8 * k);
            }
            r[k] = kHalf;
        }
        const uint32_t scales = (uint32_t)__builtin_amdgcn_readfirstlane((int)row.s.scales[tile]);
        decode_avg(mw, (int)(scales & 0xFFu), m);
        decode_sq(vw, (int)(scales >> 8), v);
    }
    for (int k = 0; k < kVec; ++k) {
        const uint32_t i = lane * kVec + k;
        if (i >= tile_n) break;
        const uint64_t e = base + i;
        float p = c.master[e];
        if (!refresh_only) {
            uint32_t cs = s;
            while (cs < c.seg_end && segs[cs].end <= e) ++cs;
            if (cs < c.seg_end && segs[cs].begin <= e) {
                const Hyper h = load_hyper<GATED>(hypers + segs[cs].hyper);
                Unscale us = us_arg;
                if constexpr (GATED) {
                    us.div_scale = h.gate_div;
                    us.inv_scale = h.gate_inv;
                    us.mode = (int)(h.gate & 0xFFu);
                }
                if (!GATED || !(h.gate >> 8)) {
                    const float g = c.grad ? Elem<GD>::to_f32(reinterpret_cast<const gscalar *>(c.grad)[e]) : 0.0f;
                    with_variant(h, us, [&](auto update) { update(g, p, m[k], v[k]); });
                    c.master[e] = p;
                    r[k] = dither_of(mix(block_key(row.s.first_block + tile, row.s.salt, h.flags >> 8) + lane * kGolden), k);
                    changed = true;
                }
            }
        }
        if constexpr (LD != ELX_NONE) {
            if (c.lowp_out) reinterpret_cast<typename Elem<LD>::scalar *>(c.lowp_out)[e] = Elem<LD>::from_f32(p);
        }
    }
    if (refresh_only || !__builtin_amdgcn_ballot_w64(changed)) return;
    int me, ve;
    uint32_t mw, vw;
    encode(m, v, r, mw, vw, me, ve);
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
        const uint32_t i = lane * kVec + k;
        if (i < tile_n) {
            mc[i] = (uint8_t)(mw >> (8 * k));
            vc[i] = (uint8_t)(vw >> (8 * k));
        }
    }
    if (lane == 0) row.s.scales[tile] = (uint16_t)(me | ve << 8);
}

template <int LD, int POLICY>
__device__ __forceinline__ void store_lowp(const ElxChunk &c, uint64_t base, const f32x4 &P) {
    if constexpr (LD != ELX_NONE) {
        if (!c.lowp_out) return;
        typedef typename Elem<LD>::vec4 lvec;
        typedef typename Elem<LD>::scalar lscalar;
        const __amdgpu_buffer_rsrc_t r = tile_rsrc(reinterpret_cast<lscalar *>(c.lowp_out) + base, kTile * sizeof(lscalar));
        lvec L;
#pragma unroll
        for (int k = 0; k < kVec; ++k) L[k] = Elem<LD>::from_f32(P[k]);
        TileIo<lvec>::template store<Aux<POLICY>::store_lowp>(r, threadIdx.x * sizeof(lvec), L);
    }
}

template <int GD, int LD, bool GATED, int POLICY>
__device__ __forceinline__ void step_tile(const ElxChunk *__restrict__ chunks, const ElxState8 *__restrict__ state,
                                          const ElxSeg *__restrict__ segs, const ElxHyper *__restrict__ hypers, Unscale us,
                                          uint32_t scalar_only) {
    const Row row = load_row(chunks + blockIdx.y, state + blockIdx.y);
    const ElxChunk &c = row.c;
    const uint32_t tile = blockIdx.x;
    const uint64_t base = (uint64_t)tile * kTile;
    if (base >= c.n_alloc) return;    // a shorter row

    typedef typename Elem<GD>::vec4 gvec;
    typedef typename Elem<GD>::scalar gscalar;
    const uint32_t lane = threadIdx.x;

    if (!scalar_only && base + kTile <= c.n_valid) {
        // the common case: a whole tile inside the valid head; all loads go out before anything is looked up
        const __amdgpu_buffer_rsrc_t pr = tile_rsrc(c.master + base, kTile * sizeof(float));
        const __amdgpu_buffer_rsrc_t mr = tile_rsrc(reinterpret_cast<uint8_t *>(c.m) + base, kTile);
        const __amdgpu_buffer_rsrc_t vr = tile_rsrc(reinterpret_cast<uint8_t *>(c.v) + base, kTile);
        // a NULL gradient is an empty buffer, which reads as zero
        const __amdgpu_buffer_rsrc_t gr =
            c.grad ? tile_rsrc(reinterpret_cast<const gscalar *>(c.grad) + base, kTile * sizeof(gscalar))
                   : tile_rsrc(c.master, 0);
        const uint32_t scales_v = row.s.scales[tile];
        const uint32_t mw = TileIo<uint32_t>::load<Aux<POLICY>::load>(mr, lane * 4);
        const uint32_t vw = TileIo<uint32_t>::load<Aux<POLICY>::load>(vr, lane * 4);
        const gvec G = TileIo<gvec>::template load<Aux<POLICY>::load>(gr, lane * sizeof(gvec));
        f32x4 P = TileIo<f32x4>::load<Aux<POLICY>::load>(pr, lane * sizeof(f32x4));
        uint32_t s = c.seg_begin, s_hi = c.seg_end;
        while (s < s_hi) {
            const uint32_t mid = (s + s_hi) >> 1;
            if (segs[mid].end > base)
                s_hi = mid;
            else
                s = mid + 1;
        }
        const bool has = s < c.seg_end;
        const uint64_t sb = has ? segs[s].begin : ~0ull;
        const uint64_t se = has ? segs[s].end : 0ull;
        if (has && sb <= base && se >= base + kTile) {
            const Hyper h = load_hyper<GATED>(hypers + segs[s].hyper);
            if constexpr (GATED) {
                us.div_scale = h.gate_div;
                us.inv_scale = h.gate_inv;
                us.mode = (int)(h.gate & 0xFFu);
                if (h.gate >> 8) {    // the step is skipped
                    store_lowp<LD, POLICY>(c, base, P);
                    return;
                }
            }
            const uint32_t word = mix(block_key(row.s.first_block + tile, row.s.salt, h.flags >> 8) + lane * kGolden);
            const uint32_t scales = (uint32_t)__builtin_amdgcn_readfirstlane((int)scales_v);
            float m[kVec], v[kVec];
            uint32_t r[kVec];
            decode_avg(mw, (int)(scales & 0xFFu), m);
            decode_sq(vw, (int)(scales >> 8), v);
            with_variant(h, us, [&](auto update) {
#pragma unroll
                for (int k = 0; k < kVec; ++k) {
                    float p = P[k];
                    update(Elem<GD>::to_f32(G[k]), p, m[k], v[k]);
                    P[k] = p;
                    r[k] = dither_of(word, k);
                }
            });
            int me, ve;
            uint32_t mo, vo;
            encode(m, v, r, mo, vo, me, ve);
            TileIo<f32x4>::store<Aux<POLICY>::store>(pr, lane * sizeof(f32x4), P);
            TileIo<uint32_t>::store<Aux<POLICY>::store>(mr, lane * 4, mo);
            TileIo<uint32_t>::store<Aux<POLICY>::store>(vr, lane * 4, vo);
            store_lowp<LD, POLICY>(c, base, P);
            if (lane == 0) row.s.scales[tile] = (uint16_t)(me | ve << 8);
            return;
        }
        if (!has || sb >= base + kTile) {    // inside the valid head but owned by no segment
            store_lowp<LD, POLICY>(c, base, P);
            return;
        }
    }

    const uint64_t left = c.n_alloc - base;
    const uint32_t tile_n = left < kTile ? (uint32_t)left : kTile;
    if (base >= c.n_valid) {    // padding: refresh only
        if (tile_n == kTile && !scalar_only) {
            if (LD == ELX_NONE || !c.lowp_out) return;
            const f32x4 P = TileIo<f32x4>::load<Aux<POLICY>::load>(tile_rsrc(c.master + base, kTile * sizeof(float)), lane * sizeof(f32x4));
            store_lowp<LD, POLICY>(c, base, P);
        } else {
            tile_any<GD, LD, GATED>(row, tile, tile_n, 0, segs, hypers, us, true);
        }
        return;
    }
    uint32_t s = c.seg_begin, s_hi = c.seg_end;
    while (s < s_hi) {
        const uint32_t mid = (s + s_hi) >> 1;
        if (segs[mid].end > base)
            s_hi = mid;
        else
            s = mid + 1;
    }
    tile_any<GD, LD, GATED>(row, tile, tile_n, s, segs, hypers, us, false);
}

template <int GD, int LD, bool GATED, int POLICY>
__global__ __launch_bounds__(kWave) void adam8_step_kernel(const ElxChunk *__restrict__ chunks,
                                                           const ElxState8 *__restrict__ state,
                                                           const ElxSeg *__restrict__ segs,
                                                           const ElxHyper *__restrict__ hypers, Unscale us,
                                                           uint32_t scalar_only) {
    step_tile<GD, LD, GATED, POLICY>(chunks, state, segs, hypers, us, scalar_only);
}

constexpr uint32_t kMaxArgHypers = 32;
struct HyperPack {
    ElxHyper h[kMaxArgHypers];
};
static_assert(offsetof(HyperPack, h) == 0, "the records start at offset 0 of the argument segment");

// hyper records in the arguments: the table the tiles read is the argument segment itself
template <int GD, int LD, int POLICY>
__global__ __launch_bounds__(kWave) void adam8_step_args_kernel(HyperPack pack, const ElxChunk *__restrict__ chunks,
                                                                const ElxState8 *__restrict__ state,
                                                                const ElxSeg *__restrict__ segs, Unscale us,
                                                                uint32_t scalar_only) {
    typedef const ElxHyper __attribute__((address_space(4))) *kernarg_hypers;
    const ElxHyper *hypers = (const ElxHyper *)(kernarg_hypers)__builtin_amdgcn_kernarg_segment_ptr();
    step_tile<GD, LD, false, POLICY>(chunks, state, segs, hypers, us, scalar_only);
}

// ---------------------------------------------------------------------------------------------
// reading and writing the state
// ---------------------------------------------------------------------------------------------

constexpr int kStateThreads = 256;    // four wavefronts, a block of the code each

template <int OD>
__device__ __forceinline__ void put_values(typename Elem<OD>::scalar *out, uint64_t at, uint64_t first, uint64_t end,
                                           const float (&x)[kVec], bool vector) {
    if (!out) return;
    if (vector && at >= first && at + kVec <= end) {
        typename Elem<OD>::vec4 w;
#pragma unroll
        for (int k = 0; k < kVec; ++k) w[k] = Elem<OD>::from_f32(x[k]);
        __builtin_nontemporal_store(w, reinterpret_cast<typename Elem<OD>::vec4 *>(out + (at - first)));
        return;
    }
#pragma unroll
    for (int k = 0; k < kVec; ++k)
        if (at + k >= first && at + k < end) out[at + k - first] = Elem<OD>::from_f32(x[k]);
}

template <int OD>
__global__ __launch_bounds__(kStateThreads) void state8_read_kernel(const uint8_t *m_codes, const uint8_t *v_codes,
                                                                    const uint16_t *__restrict__ scales, uint64_t begin,
                                                                    uint64_t n, typename Elem<OD>::scalar *m_out,
                                                                    typename Elem<OD>::scalar *v_out, uint32_t vector) {
    const uint64_t block = begin / kTile + (uint64_t)blockIdx.x * (kStateThreads / kWave) + threadIdx.x / kWave;
    const uint64_t at = block * kTile + (threadIdx.x % kWave) * kVec, end = begin + n;
    if (block * kTile >= end) return;
    uint32_t mw = 0, vw = 0;
    if (at >= begin && at + kVec <= end) {    // codes are 4-byte aligned
        if (m_out) mw = *reinterpret_cast<const uint32_t *>(m_codes + at);
        if (v_out) vw = *reinterpret_cast<const uint32_t *>(v_codes + at);
    } else {
#pragma unroll
        for (int k = 0; k < kVec; ++k)
            if (at + k >= begin && at + k < end) {
                if (m_out) mw |= (uint32_t)m_codes[at + k] << (8 * k);
                if (v_out) vw |= (uint32_t)v_codes[at + k] << (8 * k);
            }
    }
    const uint32_t s = (uint32_t)__builtin_amdgcn_readfirstlane((int)scales[block]);
    float m[kVec], v[kVec];
    decode_avg(mw, (int)(s & 0xFFu), m);
    decode_sq(vw, (int)(s >> 8), v);
    put_values<OD>(m_out, at, begin, end, m, vector);
    put_values<OD>(v_out, at, begin, end, v, vector);
}

__global__ __launch_bounds__(kStateThreads) void state8_write_kernel(const float *__restrict__ values, uint64_t n, int moment,
                                                                     uint8_t *codes, uint8_t *scales) {
    const uint64_t block = (uint64_t)blockIdx.x * (kStateThreads / kWave) + threadIdx.x / kWave;
    if (block * kTile >= n) return;
    const uint32_t lane = threadIdx.x % kWave;
    const uint64_t at = block * kTile + lane * kVec;
    float x[kVec];
    uint32_t r[kVec];
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
        x[k] = at + k < n ? values[at + k] : 0.0f;
        r[k] = kHalf;
    }
    const float none[kVec] = {};
    int me, ve;
    uint32_t mw, vw;
    if (moment)
        encode(none, x, r, mw, vw, me, ve);
    else
        encode(x, none, r, mw, vw, me, ve);
    const uint32_t w = moment ? vw : mw;
    if (at + kVec <= n) {
        *reinterpret_cast<uint32_t *>(codes + at) = w;
    } else {
#pragma unroll
        for (int k = 0; k < kVec; ++k)
            if (at + k < n) codes[at + k] = (uint8_t)(w >> (8 * k));
    }
    if (lane == 0) scales[2 * block + (moment ? 1 : 0)] = (uint8_t)(moment ? ve : me);
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------

constexpr uint32_t kUpdateFlags = ELX_FLAG_SCALAR_ONLY | ELX_FLAG_KEEP_CACHED | ELX_FLAG_KEEP_STATE_CACHED;

template <int LD>
int policy_of(uint32_t flags) {
    if (flags & ELX_FLAG_KEEP_STATE_CACHED) return kKeepState;
    if ((flags & ELX_FLAG_KEEP_CACHED) && LD != ELX_NONE) return kKeepLowp;
    return kStream;
}

struct Step {
    dim3 grid;
    uint32_t lds, flags;
    hipStream_t stream;
    const ElxChunk *chunks;
    const ElxState8 *state;
    const ElxSeg *segs;
    Unscale us;
};

template <int GD, int LD, bool GATED, int POLICY>
int launch_table(const Step &a, const ElxHyper *d_hypers) {
    hipLaunchKernelGGL((adam8_step_kernel<GD, LD, GATED, POLICY>), a.grid, dim3(kWave), a.lds, a.stream, a.chunks, a.state,
                       a.segs, d_hypers, a.us, (uint32_t)(a.flags & ELX_FLAG_SCALAR_ONLY));
    return (int)hipGetLastError();
}
template <int GD, int LD, int POLICY>
int launch_args(const Step &a, const HyperPack &pack) {
    hipLaunchKernelGGL((adam8_step_args_kernel<GD, LD, POLICY>), a.grid, dim3(kWave), a.lds, a.stream, pack, a.chunks,
                       a.state, a.segs, a.us, (uint32_t)(a.flags & ELX_FLAG_SCALAR_ONLY));
    return (int)hipGetLastError();
}

template <int GD, int LD>
int launch_types(const Step &a, const ElxHyper *d_hypers, bool gated, const HyperPack *pack) {
    constexpr int kLowp = LD != ELX_NONE ? kKeepLowp : kStream;    // no third instantiation without a low-precision copy
    switch (policy_of<LD>(a.flags)) {
        case kKeepState:
            return pack ? launch_args<GD, LD, kKeepState>(a, *pack)
                        : gated ? launch_table<GD, LD, true, kKeepState>(a, d_hypers)
                                : launch_table<GD, LD, false, kKeepState>(a, d_hypers);
        case kKeepLowp:
            return pack ? launch_args<GD, LD, kLowp>(a, *pack)
                        : gated ? launch_table<GD, LD, true, kLowp>(a, d_hypers)
                                : launch_table<GD, LD, false, kLowp>(a, d_hypers);
        default:
            return pack ? launch_args<GD, LD, kStream>(a, *pack)
                        : gated ? launch_table<GD, LD, true, kStream>(a, d_hypers)
                                : launch_table<GD, LD, false, kStream>(a, d_hypers);
    }
}

// every argument check, then the launch: a refused call launches nothing
int step(const ElxChunk *d_chunks, const ElxState8 *d_state, uint32_t n_chunks, const ElxSeg *d_segs, uint32_t n_segs,
         const ElxHyper *d_hypers, const ElxHyper *h_hypers, uint32_t n_hypers, uint64_t total_tiles, uint32_t grid_tiles,
         Unscale us, bool gated, int gd, int ld, uint32_t flags, uint32_t blocks_per_cu, void *stream) {
    if (!d_chunks || !d_state || (n_segs && (!d_segs || (!d_hypers && !h_hypers)))) return ELX_E_NULL;
    if (n_chunks == 0 || n_chunks > 65535u || total_tiles == 0 || total_tiles > 0x7FFFFFFFull || (n_segs && n_hypers == 0))
        return ELX_E_SIZE;
    if (h_hypers && n_hypers > kMaxArgHypers) return ELX_E_SIZE;
    if (grid_tiles == 0 || (uint64_t)grid_tiles * n_chunks < total_tiles) return ELX_E_TILES;
    if (!is_float_code(gd) || (ld != ELX_NONE && ld != gd)) return ELX_E_DTYPE;
    if (flags & ~kUpdateFlags) return ELX_E_RANGE;
    Step a;
    a.grid = dim3(grid_tiles, n_chunks);
    a.flags = flags;
    a.stream = (hipStream_t)stream;
    a.chunks = d_chunks;
    a.state = d_state;
    a.segs = d_segs;
    a.us = us;
    if (int rc = elx_host::occupancy_reservation(blocks_per_cu, &a.lds, kBlocksPerCu)) return rc;
    HyperPack pack = {};
    if (h_hypers) __builtin_memcpy(pack.h, h_hypers, n_hypers * sizeof(ElxHyper));
    const HyperPack *in_args = h_hypers ? &pack : nullptr;
#define ELX_CASE(G, L) \
    if (gd == G && ld == L) return launch_types<G, L>(a, d_hypers, gated, in_args);
    ELX_CASE(ELX_F32, ELX_NONE)
    ELX_CASE(ELX_F32, ELX_F32)
    ELX_CASE(ELX_F16, ELX_NONE)
    ELX_CASE(ELX_F16, ELX_F16)
    ELX_CASE(ELX_BF16, ELX_NONE)
    ELX_CASE(ELX_BF16, ELX_BF16)
#undef ELX_CASE
    return ELX_E_DTYPE;
}

constexpr uint64_t kMaxStateElems = 1ull << 33;    // of one call: a launch may have 2^32 threads, each takes four elements

}    // namespace

extern "C" {

int elx_ops_version(void) { return ELX_OPS_VERSION; }

const char *elx_ops_source_sha(void) {
#ifdef ELX_OPS_SOURCE_SHA
    return ELX_OPS_SOURCE_SHA;
#else
    return "";
#endif
}

uint32_t elx_sizeof_state8(void) { return (uint32_t)sizeof(ElxState8); }
uint32_t elx_state8_block(void) { return kTile; }

int elx_check_state8(const ElxChunk *h_chunks, const ElxState8 *h_state, uint32_t n_chunks) {
    if (!h_chunks || !h_state) return ELX_E_NULL;
    if (n_chunks == 0 || n_chunks > 65535u) return ELX_E_SIZE;
    for (uint32_t i = 0; i < n_chunks; ++i) {
        if (!h_state[i].scales) return ELX_E_NULL;
        if ((uintptr_t)h_state[i].scales & 1u) return ELX_E_ALIGN;
        if (((uintptr_t)h_chunks[i].m & 3u) || ((uintptr_t)h_chunks[i].v & 3u)) return ELX_E_ALIGN;
        if ((uint64_t)h_state[i].first_block + (h_chunks[i].n_alloc + kTile - 1) / kTile > (1ull << 32)) return ELX_E_RANGE;
    }
    return 0;
}

int elx_adam8_step_mt(const ElxChunk *d_chunks, const ElxState8 *d_state, uint32_t n_chunks, const ElxSeg *d_segs,
                      uint32_t n_segs, const ElxHyper *d_hypers, uint32_t n_hypers, uint64_t total_tiles,
                      uint32_t grid_tiles_per_chunk, float div_scale, int grad_dtype, int lowp_dtype, uint32_t flags,
                      uint32_t blocks_per_cu, void *stream) {
    return step(d_chunks, d_state, n_chunks, d_segs, n_segs, d_hypers, nullptr, n_hypers, total_tiles, grid_tiles_per_chunk,
                elx_host::unscale_of(div_scale), false, grad_dtype, lowp_dtype, flags, blocks_per_cu, stream);
}

int elx_adam8_step_args_mt(const ElxChunk *d_chunks, const ElxState8 *d_state, uint32_t n_chunks, const ElxSeg *d_segs,
                           uint32_t n_segs, const ElxHyper *h_hypers, uint32_t n_hypers, uint64_t total_tiles,
                           uint32_t grid_tiles_per_chunk, float div_scale, int grad_dtype, int lowp_dtype, uint32_t flags,
                           uint32_t blocks_per_cu, void *stream) {
    if (!h_hypers) return ELX_E_NULL;
    if (n_hypers == 0) return ELX_E_SIZE;
    return step(d_chunks, d_state, n_chunks, d_segs, n_segs, nullptr, h_hypers, n_hypers, total_tiles, grid_tiles_per_chunk,
                elx_host::unscale_of(div_scale), false, grad_dtype, lowp_dtype, flags, blocks_per_cu, stream);
}

int elx_adam8_step_gated_mt(const ElxChunk *d_chunks, const ElxState8 *d_state, uint32_t n_chunks, const ElxSeg *d_segs,
                            uint32_t n_segs, const ElxHyper *d_hypers, uint32_t n_hypers, uint64_t total_tiles,
                            uint32_t grid_tiles_per_chunk, int grad_dtype, int lowp_dtype, uint32_t flags,
                            uint32_t blocks_per_cu, void *stream) {
    return step(d_chunks, d_state, n_chunks, d_segs, n_segs, d_hypers, nullptr, n_hypers, total_tiles, grid_tiles_per_chunk,
                elx_host::unscale_of(-1.0f), true, grad_dtype, lowp_dtype, flags, blocks_per_cu, stream);
}

int elx_state8_read(const uint8_t *m_codes, const uint8_t *v_codes, const uint16_t *scales, uint64_t begin, uint64_t n,
                    void *m_out, void *v_out, int out_dtype, void *stream) {
    if (!scales || (!m_out && !v_out) || (m_out && !m_codes) || (v_out && !v_codes)) return ELX_E_NULL;
    if (out_dtype != ELX_F32 && out_dtype != ELX_BF16) return ELX_E_DTYPE;
    if (n == 0 || n > kMaxStateElems || begin > (1ull << 40)) return ELX_E_SIZE;
    const uintptr_t outs = (uintptr_t)m_out | (uintptr_t)v_out, es = elem_size(out_dtype);
    if ((outs & (es - 1)) || ((uintptr_t)scales & 1u) || (((uintptr_t)m_codes | (uintptr_t)v_codes) & 3u)) return ELX_E_ALIGN;
    const uint32_t vector = begin % kVec == 0 && outs % (kVec * es) == 0;
    const uint64_t blocks = (begin + n + kTile - 1) / kTile - begin / kTile;
    const dim3 grid((uint32_t)((blocks + kStateThreads / kWave - 1) / (kStateThreads / kWave)));
    if (out_dtype == ELX_F32)
        hipLaunchKernelGGL((state8_read_kernel<ELX_F32>), grid, dim3(kStateThreads), 0, (hipStream_t)stream, m_codes, v_codes,
                           scales, begin, n, (float *)m_out, (float *)v_out, vector);
    else
        hipLaunchKernelGGL((state8_read_kernel<ELX_BF16>), grid, dim3(kStateThreads), 0, (hipStream_t)stream, m_codes, v_codes,
                           scales, begin, n, (uint16_t *)m_out, (uint16_t *)v_out, vector);
    return (int)hipGetLastError();
}

int elx_state8_write(const float *values, uint64_t n, int moment, uint8_t *codes, uint16_t *scales, void *stream) {
    if (!values || !codes || !scales) return ELX_E_NULL;
    if (moment != 0 && moment != 1) return ELX_E_RANGE;
    if (n == 0 || n > kMaxStateElems) return ELX_E_SIZE;
    if (((uintptr_t)values & 3u) || ((uintptr_t)codes & 3u) || ((uintptr_t)scales & 1u)) return ELX_E_ALIGN;
    const uint64_t blocks = (n + kTile - 1) / kTile;
    const dim3 grid((uint32_t)((blocks + kStateThreads / kWave - 1) / (kStateThreads / kWave)));
    hipLaunchKernelGGL(state8_write_kernel, grid, dim3(kStateThreads), 0, (hipStream_t)stream, values, n, moment, codes,
                       reinterpret_cast<uint8_t *>(scales));
    return (int)hipGetLastError();
}

}    // extern "C"
