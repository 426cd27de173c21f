// HIPCC_FLAGS: -fno-slp-vectorize -Xclang -target-feature -Xclang -packed-fp32-ops
// Attention over contexts: every query of a sample attends to `Np` keys that all samples share (the prefix) and to the sample's own keys,
// of which the first lens[b] exist (fewer where a key mask is given).  fp16 / bf16 storage, head widths 8..128 (multiples of 8), H query heads on Hk key heads.
//
//   s = scale q k^T over the keys that exist,  p = exp(s - max),  o = sum p v / sum p      (no key: o = 0, lse = -inf)
//
// One pass over the keys with a running maximum and sum, fp32 accumulators.  S is computed transposed (A = K rows out of LDS, B = Q^T in registers), so
// a lane owns one query column: its maximum, sum and rescaling are lane-local but for one exchange between the two lane halves, and its
// probabilities already lie in the order in which the second product takes its B operand (the k order of an MFMA is free as long as A
// uses the same: V^T is fetched with the transpose read in that order).  Keys that do not exist are zeroed while they are staged (a NaN
// there reaches nothing) and their scores are -inf.
//
// What bounds the products: no pipe alone.  On full grids the matrix pipes are busy 37 to 56 % of a SIMD's clocks and vector instructions (the softmax, roundings,
// addresses) are issued in 28 to 59 %, LDS has no bank conflicts (counters, all keys in use: k_ctx_attn 14 x 5 x 4096 x 8192 of 64 41 and 59 %, 2 x 16 x 4096 x 4096 of 128
// 43 and 37, k_ctx_bwd_q 56 and 38, k_ctx_bwd_kv 37 and 28): two or three waves a SIMD do not cover each other's waits for LDS and between the products.
// A wave's 32 columns use every A operand that LDS gives (1 KB, 8 clocks of its 128 B) for one MFMA of 32 clocks; 64 columns would halve the reads, but their
// accumulators leave one wave a SIMD (a version of many_rows, slower).  Rates below are of the products that the formulas need, with all keys in use.
#include "common.h"

namespace {

typedef unsigned short u16;
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4* lds4;
template <int V> struct Const { static constexpr int value = V; };

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

template <bool BF> __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {      // 32x32x16
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <bool BF> __device__ __forceinline__ unsigned pack2(float lo, float hi) {           // one rounding to nearest even each
    if constexpr (BF) return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{lo, hi}, b2));
    else return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{lo, hi}, h2));
}
// acc + a.lo b.lo + a.hi b.hi
template <bool BF> __device__ __forceinline__ float dot2(unsigned a, unsigned b, float acc) {
    if constexpr (BF) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, a), __builtin_bit_cast(b2, b), acc, false);
    else return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, a), __builtin_bit_cast(h2, b), acc, false);
}
__device__ __forceinline__ f32x16 zero16() { return f32x16{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}; }
// the same value in both lane halves: max / sum over lanes l and l + 32
__device__ __forceinline__ float half_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// LDS tile [row][DP] of 16-bit values without padding.  16-byte slot s of row r lies at slot s ^ swz(r): a 16-lane row read (16 rows, one
// slot) and a transpose read (4 rows of one 64-byte piece per lane group, two groups side by side) both touch each of the 64 banks once.
template <int DP> __device__ __forceinline__ int swz(int r) {
    if constexpr (DP == 64) return ((r & 2) << 1) | ((r >> 2) & 3);
    else if constexpr (DP == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
    else return (r >> 2) & 3;
}
template <int DP> __device__ __forceinline__ int slot_at(int r, int s) { return r * DP + ((s ^ swz<DP>(r)) << 3); }

// A fragment of the transposed tile: lane (l31, hi) gets column c0 + l31 of rows r0 + 4 hi + 0..3 and r0 + 8 + 4 hi + 0..3, r0 a multiple of 16 --
// the rows that an accumulator's registers 8 s .. 8 s + 7 hold in that lane half.
template <int DP> __device__ __forceinline__ u32x4 read_tr(const u16* t, int r0, int c0, int lane) {
    const int hi = lane >> 5, r = r0 + 4 * hi + ((lane & 15) >> 2);
    const int slot = (c0 >> 3) + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1), in = (lane & 1) * 4;
    struct { s16x4 a, b; } v = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(t + slot_at<DP>(r, slot) + in)),
                                __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(t + slot_at<DP>(r + 8, slot) + in))};
    return __builtin_bit_cast(u32x4, v);
}
template <int DP> __device__ __forceinline__ u32x4 read_row(const u16* t, int r, int slot) { return *reinterpret_cast<const u32x4*>(t + slot_at<DP>(r, slot)); }

// Fetching of tiles of 64 rows straight into LDS (16 bytes a lane, four waves): lane i of piece w + 4 j fills 16-byte place (w + 4 j) 64 + i of the tile, so it
// asks for the slot that belongs there.  What does not exist is asked for beyond the buffer's end and arrives as zeros.
//
// The fetch is spelled out: of one that it can see the compiler assumes that any LDS read might want its data and waits for it, the next tile's
// fetches too.  It has no register result; landed() waits for it.  (s_nop 4: an SGPR that a vector instruction has just written, and M0, are settled;
// nothing else in this file keeps a value in M0.)
constexpr unsigned BEYOND = 0xF0000000u;
struct Span {
    u32x4 r;                   // buffer resource: address, no stride, 0xE0000000 bytes
    __device__ __forceinline__ explicit Span(const u16* at) {
        const unsigned long long a = (unsigned long long)at;
        r = u32x4{(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)a), (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32)) & 0xffffu, 0xE0000000u, 0x00020000u};
    }
    __device__ __forceinline__ void fetch(u16* lds, unsigned off, int step) const {
#if defined(__HIP_DEVICE_COMPILE__)
        const int m0 = __builtin_amdgcn_readfirstlane((int)(unsigned)(unsigned long long)lds);     // the low half of a generic LDS address is its offset
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(m0), "v"(off), "s"(r), "s"(step));
#endif
    }
};
template <int DP> struct Fetch {
    static constexpr int SL = DP / 8, N = 64 * SL / 256, M = 256 % SL ? N : 1;      // M = 1: a lane's places differ by whole rows that the swizzle does not see
    unsigned off[M];
    static __device__ __forceinline__ int row(int tid, int j) { return M == 1 ? tid / SL + j * (256 / SL) : (tid + 256 * j) / SL; }
    __device__ __forceinline__ void init(int tid, long long step, int d) {           // step: elements from row to row (64 of them below 2^31 bytes)
#pragma unroll
        for (int j = 0; j < M; ++j) {
            const int r = row(tid, j), c = (((tid + 256 * j) % SL) ^ swz<DP>(r)) * 8;
            off[j] = c < d ? (unsigned)(r * (int)step + c) * 2u : BEYOND;
        }
    }
    // the tile at `at`; rows of it that exist: live
    __device__ __forceinline__ void tile(const u16* at, long long step, unsigned long long live, u16* lds, int tid, int wave) const {
        const Span span(at);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const unsigned o = off[M == 1 ? 0 : j];
            span.fetch(lds + (wave + 4 * j) * 512, live == ~0ull || ((live >> row(tid, j)) & 1) ? o : BEYOND, M == 1 ? j * (512 / SL) * (int)step : 0);
        }
    }
};
// this wave's fetches and writes are in LDS; the barrier makes all of them visible
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

struct AttnArgs {
    const u16 *q, *kp, *vp, *k, *v;
    long long q_b, q_n, q_h, kp_n, kp_h, vp_n, vp_h, k_b, k_n, k_h, v_b, v_n, v_h;      // element strides
    const int* lens;
    const unsigned char* mask;
    long long mask_b;
    u16 *o, *o_lo;             // [B][Nq][H][d]; o_lo (or null): what the rounding of o left, for the backward pass
    float* lse;                // [B][H][Nq] or null
    float *po, *pml;           // partial results: [part][B * Nq * H][d], [..][2] = (maximum in log2 units, sum)
    int B, Nq, Np, Nk, H, Hk, G, d, causal;
    float c;                   // scale * log2 e
};
// A share of a launch's blocks: row tiles x runs of key tiles x key heads (x samples).  A call has up to two of them.
struct Deal {
    int blocks, xtiles;        // row tiles of a key head
    int splits, per_split;     // key tiles are dealt out in runs of per_split
    int part0;                 // index of its first partial result
    int stacked;               // rows run over (sample, query, head of the group) and see the prefix alone; else the rows of one sample
    int np;                    // prefix keys that it visits
};

// One row (query, head) per accumulator column.  Rows of a key head: r = (sample, query, head of its group), heads fastest.
struct Row {
    int b, qi, h;
    bool on;
};
__device__ __forceinline__ Row row_of(const AttnArgs& p, int b, int hk, bool stacked, int r, int rows) {      // (divisions only where a call has groups or stacked rows)
    Row x;
    x.on = r < rows;
    unsigned i = x.on ? r : rows - 1;
    x.b = b;
    if (stacked) {
        const unsigned per = p.Nq * p.G, bb = i / per;
        x.b += bb;
        i -= bb * per;
    }
    x.qi = i;
    x.h = hk;
    if (p.G > 1) {
        x.qi = i / (unsigned)p.G;
        x.h = hk * p.G + i - x.qi * p.G;
    }
    return x;
}

// Blocks reach the 8 XCDs round-robin by their index: every XCD gets one contiguous run of the (sample, key head, split, row tile) space, so the row
// tiles that read the same keys share them through one L2.  Samples are outermost: of a few samples of unequal length the short ones' XCDs are done first.
__device__ __forceinline__ unsigned swizzled(unsigned i, unsigned tot) {
    const unsigned q = tot / 8, r = tot % 8, xcd = i % 8;
    return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + i / 8;
}
__device__ __forceinline__ void block_of(int xtiles, int& y, int& xt) {
    const unsigned id = swizzled(blockIdx.x, gridDim.x);
    y = (int)(id / xtiles);
    xt = (int)(id % xtiles);
}
struct Place {
    int b, hk, split, xt, len, rows;   // len: own keys
};
__device__ __forceinline__ Place place_of(const AttnArgs& p, const Deal& w, unsigned i) {
    Place x;
    const unsigned id = swizzled(i, w.blocks);
    x.xt = id % w.xtiles;
    unsigned y = id / w.xtiles;
    x.split = y % w.splits;
    y /= w.splits;
    x.hk = y % p.Hk;
    x.b = y / p.Hk;
    x.rows = (w.stacked ? p.B : 1) * p.Nq * p.G;                       // below 2^31 (checked)
    x.len = w.stacked ? 0 : (p.lens ? max(0, min(p.lens[x.b], p.Nk)) : p.Nk);
    return x;
}

// Q^T of one row as B operands: lane (l31, hi) holds d = 16 s + 8 hi + 0..7 of its row
template <int DP> __device__ __forceinline__ void load_q(const AttnArgs& p, const Row& x, int hi, u32x4 (&f)[DP / 16]) {
    const u16* qp = p.q + x.b * p.q_b + x.qi * p.q_n + x.h * p.q_h;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const int at = s * 16 + hi * 8;
        f[s] = *reinterpret_cast<const u32x4*>(qp + (at < p.d ? at : 0));
    }
    if (p.d < DP)
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
            if (s * 16 + hi * 8 >= p.d) f[s] = u32x4{0u, 0u, 0u, 0u};
}

// 32 columns n * 32 .. of one row out of its accumulator, times f, as 16-byte pieces: the lane halves hold the rows 4 hi .. of every
// 8 channels, one exchange of two registers gives each half 8 neighbouring channels.  lo: what the rounding left.  All lanes call it.
template <bool BF> __device__ __forceinline__ float value_of(unsigned x, int half) {
    const unsigned short w = half ? x >> 16 : x & 0xffffu;
    return BF ? __uint_as_float((unsigned)w << 16) : (float)__builtin_bit_cast(_Float16, w);
}
template <bool BF> __device__ __forceinline__ unsigned left2(float a, float b) {
    const unsigned x = pack2<BF>(a, b);
    return pack2<BF>(a - value_of<BF>(x, 0), b - value_of<BF>(x, 1));
}
// channels 16 g + 8 hi .. + 7 of a block of 32
template <bool BF, bool LEFT = false> __device__ __forceinline__ u32x4 eight(const f32x16& a, float f, int g) {
    auto two = [&](int r) __attribute__((always_inline)) { return LEFT ? left2<BF>(a[r] * f, a[r + 1] * f) : pack2<BF>(a[r] * f, a[r + 1] * f); };
    const auto x = __builtin_amdgcn_permlane32_swap(two(8 * g), two(8 * g + 4), false, false);
    const auto y = __builtin_amdgcn_permlane32_swap(two(8 * g + 2), two(8 * g + 6), false, false);
    return u32x4{x[0], y[0], x[1], y[1]};
}
template <bool BF, bool LEFT = false> __device__ __forceinline__ void store_row(u16* row, const f32x16& a, float f, int n, int hi, int d, bool on) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const int c = n * 32 + 16 * g + 8 * hi;
        const u32x4 x = eight<BF, LEFT>(a, f, g);
        if (on && c < d) *reinterpret_cast<u32x4*>(row + c) = x;
    }
}

// One step of the running softmax on a block of 32 scores: probabilities p = exp2(s c - m) as B operands, their sum of this lane half into l.  m (log2 units)
// is moved only where it has to be: for a row's first key, and where a half's sum of 16 probabilities passes 2^12 (fp16 holds 2^16) -- the maximum,
// the rescaling and the exchange between the lane halves are then done and the probabilities taken anew; otherwise the scores are touched once.
template <bool BF, int ND> __device__ __forceinline__ void soften(const f32x16& s, float c, float& m, float& l, f32x16 (&acc)[ND], u32x4 (&fp)[2]) {
    float sum;
    auto take = [&](float ref) __attribute__((always_inline)) {
        float a[2] = {0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[r], c, -ref)), p1 = __builtin_amdgcn_exp2f(fmaf(s[r + 1], c, -ref));
            fp[r >> 3][(r >> 1) & 3] = pack2<BF>(p0, p1);             // the one rounding of the probabilities
            a[0] += p0;
            a[1] += p1;
        }
        sum = a[0] + a[1];
    };
    const bool none = m == -INFINITY;
    take(none ? 0.f : m);
    if (__builtin_expect(__any(none || !(sum <= 4096.f)), 0)) {
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        const float m_new = fmaxf(m, half_max(mx) * c);
        const float ref = m_new == -INFINITY ? 0.f : m_new;           // still no key: every exp2 gives 0
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
        l *= alpha;
#pragma unroll
        for (int n = 0; n < ND; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[n][r] *= alpha;
        m = m_new;
        take(ref);
    }
    l += sum;
}

// -inf into the scores of keys that do not exist (bits) or lie behind lim (in this lane's numbering)
__device__ __forceinline__ void hide(f32x16& s, unsigned bits, int lim, int hi) {
    bits >>= 4 * hi;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int at = (r & 3) + 8 * (r >> 2);
        if (!((bits >> at) & 1u) || at > lim) s[r] = -INFINITY;
    }
}

// Many rows: the block's four waves own 32 rows each and share key tiles of 64 in LDS, fetched one tile ahead.  14 x 5 heads x 4096 rows x 8192 keys of 64
// (fp16) 725 to 780 us one after the other, 775 to 830 TFLOP/s at the clock that the power limit leaves; 2 x 16 heads x 4096 x 4096 of 128 (bf16) 299 us, 920 TFLOP/s;
// a large library product reaches 1250 on the same card.  8 samples' prompts of 512 behind 4096 shared keys, causal, 32 heads of 128 on 8 (bf16): 359 us, 815.
// Single tokens of 64 samples over a prefix of 16384, 32 heads of 128 on 8: 38 us alone, 455 TFLOP/s -- 8 tiles a block, too few to hide a block's
// start and its partial results (68 MB in all).
template <bool BF, int DP> __device__ __forceinline__ void many_rows(const AttnArgs& p, const Deal& w, unsigned block, u16* lds) {
    constexpr int KT = 64, ND = DP / 32, TILE = KT * DP, BR = 128;
    u16 *sK = lds, *sV = lds + 2 * TILE;                              // two buffers each
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, hi = lane >> 5;
    const Place at = place_of(p, w, block);
    const int r0 = at.xt * BR;
    const Row row = row_of(p, at.b, at.hk, w.stacked, r0 + wave * 32 + l31, at.rows);
    u32x4 fq[DP / 16];
    load_q<DP>(p, row, hi, fq);
    const int last_r = min(r0 + BR, at.rows) - 1;
    const int seen = p.causal ? max(0, min(at.len, at.len - p.Nq + 1 + last_r / p.G)) : at.len;      // own keys that the block's last row sees
    const int all_see = p.causal ? at.len - p.Nq + 1 + r0 / p.G : at.len;                             // own keys that every row sees
    const int T0 = (w.np + KT - 1) / KT, T1 = (seen + KT - 1) / KT;
    const int tb = min(at.split * w.per_split, T0 + T1), te = w.splits == 1 ? T0 + T1 : min(tb + w.per_split, T0 + T1);

    unsigned long long live = 0;                                      // keys of the fetched tile that exist
    const u16 *kown = p.k + at.b * p.k_b + at.hk * p.k_h, *vown = p.v + at.b * p.v_b + at.hk * p.v_h;
    const u16 *kpre = p.kp + at.hk * p.kp_h, *vpre = p.vp + at.hk * p.vp_h;
    const unsigned char* mrow = p.mask ? p.mask + at.b * p.mask_b : nullptr;
    Fetch<DP> fk, fv;
    bool prefix = tb < T0;
    fk.init(tid, prefix ? p.kp_n : p.k_n, p.d);
    fv.init(tid, prefix ? p.vp_n : p.v_n, p.d);
    auto fetch = [&](int t, int buf) __attribute__((always_inline)) {
        if (prefix && t >= T0) {
            prefix = false;
            fk.init(tid, p.k_n, p.d);
            fv.init(tid, p.v_n, p.d);
        }
        const int k0 = (prefix ? t : t - T0) * KT, n = (prefix ? w.np : seen) - k0;
        const long long kn = prefix ? p.kp_n : p.k_n, vn = prefix ? p.vp_n : p.v_n;
        live = n >= KT ? ~0ull : (1ull << n) - 1;
        if (!prefix && mrow) live = __ballot(lane < n && mrow[k0 + min(lane, n - 1)]);
        fk.tile((prefix ? kpre : kown) + k0 * kn, kn, live, sK + buf * TILE, tid, wave);
        fv.tile((prefix ? vpre : vown) + k0 * vn, vn, live, sV + buf * TILE, tid, wave);
    };
    f32x16 acc[ND];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int n = 0; n < ND; ++n) acc[n] = zero16();
    if (tb < te) fetch(tb, 0);
    landed();
    auto work = [&](auto which, int t) __attribute__((always_inline)) {                              // the buffer is a constant of the code: every LDS address is one register and an immediate
        constexpr int buf = decltype(which)::value;
        const u16* tk = sK + buf * TILE;
        const unsigned long long now = live;
        if (t + 1 < te) fetch(t + 1, buf ^ 1);
        const int k0 = (t >= T0 ? t - T0 : t) * KT;
        const bool edge = p.causal && t >= T0 && k0 + KT > all_see;
        // both halves' scores first: the matrix pipe works on the second while the first becomes probabilities
        f32x16 s[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < DP / 16; ++e) s[j] = mfma<BF>(read_row<DP>(tk, j * 32 + l31, e * 2 + hi), fq[e], e ? s[j] : zero16());
        if (now != ~0ull || edge)
#pragma unroll
            for (int j = 0; j < 2; ++j) hide(s[j], (unsigned)(now >> (32 * j)), edge ? at.len - p.Nq + row.qi - k0 - 32 * j - 4 * hi : 1 << 30, hi);
        auto half = [&](auto which_half) __attribute__((always_inline)) {
            constexpr int j = decltype(which_half)::value;
            u32x4 fp[2];
            soften<BF, ND>(s[j], p.c, m, l, acc, fp);
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int n = 0; n < ND; ++n) acc[n] = mfma<BF>(read_tr<DP>(sV + buf * TILE, j * 32 + e * 16, n * 32, lane), fp[e], acc[n]);
        };
        half(Const<0>{});
        half(Const<1>{});
        landed();
    };
    for (int t = tb; t < te; t += 2) {
        work(Const<0>{}, t);
        if (t + 1 < te) work(Const<1>{}, t + 1);
    }
    const long long total = (long long)p.B * p.Nq * p.H, part = w.part0 + at.split;
    l = half_sum(l);
    const long long id = ((long long)row.b * p.Nq + row.qi) * p.H + row.h;
    const float inv = l > 0.f ? __builtin_amdgcn_rcpf(l) : 0.f;
#pragma unroll
    for (int n = 0; n < ND; ++n) {
        if (!p.po) {
            store_row<BF>(p.o + id * p.d, acc[n], inv, n, hi, p.d, row.on);
            if (p.o_lo) store_row<BF, true>(p.o_lo + id * p.d, acc[n], inv, n, hi, p.d, row.on);
        } else if (row.on) {
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int c = n * 32 + 2 * r + 4 * hi;
                if (c < p.d) *reinterpret_cast<f32x4*>(p.po + (part * total + id) * p.d + c) = f32x4{acc[n][r], acc[n][r + 1], acc[n][r + 2], acc[n][r + 3]};
            }
        }
    }
    if (hi == 0 && row.on) {
        if (p.po) *reinterpret_cast<f32x2*>(p.pml + (part * total + id) * 2) = f32x2{m, l};
        else if (p.lse) p.lse[((long long)row.b * p.H + row.h) * p.Nq + row.qi] = (m + __builtin_amdgcn_logf(l)) * LN2;
    }
}

// Few rows (at most 32 per key head): the keys are what has to be read, so every wave walks over its own runs of 32 of them with all rows as
// columns, no barrier in the loop.  64 samples of one query over 2000 keys, 16 heads of 64 (fp16): 111 us, 4.7 TB/s; 32 over 5000, 8 heads of 128: 124 us,
// 5.3 TB/s, the rate of a large copy (K read row by row into the operands, past LDS: 128 and 136 us, every line fetched four times).  K and V pass through a piece of LDS that only this wave uses (read whole rows at a time).
// The next 32 keys are in flight while these are worked on; the four waves' results are merged at the end.
template <bool BF, int DP> __device__ __forceinline__ void few_rows(const AttnArgs& p, const Deal& w, unsigned block, u16* lds) {
    constexpr int SL = DP / 8, NV = 32 * SL / 64, ND = DP / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, hi = lane >> 5;
    u16 *sK = lds + wave * 64 * DP, *sV = sK + 32 * DP;
    const Place at = place_of(p, w, block);
    const int rows = at.rows;
    const Row row = row_of(p, at.b, at.hk, w.stacked, l31, rows);
    u32x4 fq[DP / 16];
    load_q<DP>(p, row, hi, fq);
    const int len = at.len;                                           // causal: the last row sees all of them
    const int T0 = (w.np + 127) / 128, T1 = (len + 127) / 128;
    const int tb = min(at.split * w.per_split, T0 + T1), te = w.splits == 1 ? T0 + T1 : min(tb + w.per_split, T0 + T1);
    u32x4 rk[NV], rv[NV];
    const u16 *kown = p.k + at.b * p.k_b + at.hk * p.k_h, *vown = p.v + at.b * p.v_b + at.hk * p.v_h;
    const unsigned char* mrow = p.mask ? p.mask + at.b * p.mask_b : nullptr;
    // the tile's first key; a tile's last runs may lie behind the segment
    auto first = [&](int t) __attribute__((always_inline)) { return (t >= T0 ? t - T0 : t) * 128 + wave * 32; };
    auto load = [&](int t) __attribute__((always_inline)) {
        const bool own = t >= T0;
        const int n = own ? len : w.np, k0 = first(t);
        const u16 *kb = own ? kown : p.kp + at.hk * p.kp_h, *vb = own ? vown : p.vp + at.hk * p.vp_h;
        const long long kn = own ? p.k_n : p.kp_n, vn = own ? p.v_n : p.vp_n;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int id = lane + 64 * i, c = id % SL * 8, r = min(k0 + id / SL, n - 1);
            rk[i] = *reinterpret_cast<const u32x4*>(kb + r * kn + (c < p.d ? c : 0));
            rv[i] = *reinterpret_cast<const u32x4*>(vb + r * vn + (c < p.d ? c : 0));
        }
    };
    auto exists = [&](int t) -> unsigned {
        const bool own = t >= T0;
        const int n = own ? len : w.np, key = first(t) + l31;
        return (unsigned)__ballot(key < n && (!own || !mrow || mrow[min(key, n - 1)]));
    };
    f32x16 acc[ND];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[n][r] = 0.f;
    unsigned bits = 0;
    if (tb < te) {
        load(tb);
        bits = exists(tb);
    }
    for (int t = tb; t < te; ++t) {
        const unsigned now = bits;
        const bool more = t + 1 < te;
        if (more) bits = exists(t + 1);
#pragma unroll
        for (int i = 0; i < NV; ++i) {                                // keys that do not exist and channels behind d are zero
            const int id = lane + 64 * i, r = id / SL, slot = id % SL;
            if (slot * 8 >= p.d || !((now >> r) & 1u)) rk[i] = rv[i] = u32x4{0u, 0u, 0u, 0u};
            *reinterpret_cast<u32x4*>(sK + slot_at<DP>(r, slot)) = rk[i];
            *reinterpret_cast<u32x4*>(sV + slot_at<DP>(r, slot)) = rv[i];
        }
        if (more) load(t + 1);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");        // the other lanes' rows are in place (a wave's LDS operations keep their order)
        __builtin_amdgcn_wave_barrier();
        f32x16 s = zero16();
#pragma unroll
        for (int e = 0; e < DP / 16; ++e) s = mfma<BF>(read_row<DP>(sK, l31, e * 2 + hi), fq[e], s);
        const int k0 = first(t);
        const bool edge = p.causal && t >= T0 && k0 + 32 > len - p.Nq + 1;
        if (now != ~0u || edge) hide(s, now, edge ? len - p.Nq + row.qi - k0 - 4 * hi : 1 << 30, hi);
        u32x4 fp[2];
        soften<BF, ND>(s, p.c, m, l, acc, fp);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int n = 0; n < ND; ++n) acc[n] = mfma<BF>(read_tr<DP>(sV, e * 16, n * 32, lane), fp[e], acc[n]);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");        // ... and read before the next ones replace them
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    // maxima and sums first, then the accumulators, fp32 [wave][row][DP + 4]; rows that do not exist are left out
    float* sm = reinterpret_cast<float*>(lds);                        // [4][32] maxima, [4][32] sums
    float* so = sm + 256;
    constexpr int LD = DP + 4;
    l = half_sum(l);
    if (hi == 0) {
        sm[wave * 32 + l31] = m;
        sm[128 + wave * 32 + l31] = l;
    }
    if (l31 < rows)
#pragma unroll
        for (int n = 0; n < ND; ++n)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *reinterpret_cast<f32x4*>(so + (wave * 32 + l31) * LD + n * 32 + 2 * r + 4 * hi) = f32x4{acc[n][r], acc[n][r + 1], acc[n][r + 2], acc[n][r + 3]};
    __syncthreads();
    const long long total = (long long)p.B * p.Nq * p.H, part = w.part0 + at.split;
    const int rr = tid >> 3;
    const Row x = row_of(p, at.b, at.hk, w.stacked, rr, rows);
    if (!x.on) return;
    float mm = -INFINITY, ll = 0.f, f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) mm = fmaxf(mm, sm[i * 32 + rr]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = mm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[i * 32 + rr] - mm);
        ll += f[i] * sm[128 + i * 32 + rr];
    }
    const long long id = ((long long)x.b * p.Nq + x.qi) * p.H + x.h;
    const float inv = ll > 0.f ? __builtin_amdgcn_rcpf(ll) : 0.f;
    for (int c = (tid & 7) * 4; c < p.d; c += 32) {
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 t = *reinterpret_cast<const f32x4*>(so + (i * 32 + rr) * LD + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] += f[i] * t[e];
        }
        if (p.po) *reinterpret_cast<f32x4*>(p.po + (part * total + id) * p.d + c) = a;
        else {
            *reinterpret_cast<u32x2*>(p.o + id * p.d + c) = u32x2{pack2<BF>(a[0] * inv, a[1] * inv), pack2<BF>(a[2] * inv, a[3] * inv)};
            if (p.o_lo) *reinterpret_cast<u32x2*>(p.o_lo + id * p.d + c) = u32x2{left2<BF>(a[0] * inv, a[1] * inv), left2<BF>(a[2] * inv, a[3] * inv)};
        }
    }
    if ((tid & 7) == 0) {
        if (p.po) *reinterpret_cast<f32x2*>(p.pml + (part * total + id) * 2) = f32x2{mm, ll};
        else if (p.lse) p.lse[((long long)x.b * p.H + x.h) * p.Nq + x.qi] = (mm + __builtin_amdgcn_logf(ll)) * LN2;
    }
}

constexpr int lds_many(int DP) { return 4 * 64 * DP; }                                             // in 16-bit units
constexpr int lds_few(int DP) { return (256 + 128 * (DP + 4)) * 2; }
constexpr int larger(int a, int b) { return a > b ? a : b; }

// first: the stacked prefix rows (may be none), second: the samples' own rows
enum { MANY, FEW, MIXED };                                                                         // MIXED: many stacked rows, few own rows
template <bool BF, int DP, int MODE> __global__ void __launch_bounds__(256, MODE == MANY && DP == 64 ? 3 : 2) k_ctx_attn(AttnArgs p, Deal first, Deal second) {
    __shared__ __attribute__((aligned(16))) u16 lds[MODE == MANY ? lds_many(DP) : MODE == FEW ? lds_few(DP) : larger(lds_many(DP), lds_few(DP))];
    const bool one = (int)blockIdx.x < first.blocks;
    const Deal& w = one ? first : second;
    const unsigned block = one ? blockIdx.x : blockIdx.x - first.blocks;
    if (MODE == MANY || (MODE == MIXED && one)) many_rows<BF, DP>(p, w, block, lds);
    else few_rows<BF, DP>(p, w, block, lds);
}

// A context of at most 96 keys and many rows: the rows are what has to be read and written.  The block keeps every key of its key head in LDS and each wave
// walks over tiles of 32 rows by itself, the next tile's queries in flight; all scores of a row are there at once, so nothing is rescaled.  Keys that do not
// exist enter through the first product's accumulator, which starts at -inf for them (0 for the others).  28 x 4096 rows x 77 keys, 5 heads of 64 (fp16):
// 33.5 to 41 us with fresh inputs (3.7 to 4.5 TB/s; a copy of the same bytes 29).  96 keys leave registers for three waves a SIMD.
constexpr int SHORT = 96;
template <bool BF, int DP> __global__ void __launch_bounds__(256, DP == 64 ? 3 : 2) k_ctx_short(AttnArgs p, int chunks, int per_chunk) {
    constexpr int SL = DP / 8, NST = (SHORT * SL + 255) / 256, ND = DP / 32;
    __shared__ __attribute__((aligned(16))) u16 sK[SHORT * DP], sV[SHORT * DP];
    __shared__ __attribute__((aligned(16))) float sE[SHORT];
    // A lane computes one row, but memory wants whole rows an instruction (each lane its own row, 32 bytes of a line at a time: 28 x 4096 x 77 keys 49 us for
    // 36, 33 keys 46 for 31): queries and results change places through a piece of LDS of this wave's own.  Heads over 96 wide leave no room for
    // it beside a second block.
    constexpr bool STAGED = DP <= 96;
    __shared__ __attribute__((aligned(16))) u16 sT[STAGED ? 4 * 32 * DP : 8];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, hi = lane >> 5;
    int y, chunk;
    block_of(chunks, y, chunk);
    const int hk = y % p.Hk, b = y / p.Hk, rows = p.Nq * p.G;
    const int t1 = min((chunk + 1) * per_chunk, (rows + 31) / 32), t0 = chunk * per_chunk + wave;
    const bool plain = p.G == 1;                                     // whole tiles without groups: uniform base, offsets below 2^32
    const u16* q0 = p.q + b * p.q_b + hk * p.q_h;
    u16 *o0 = p.o + ((long long)b * p.Nq * p.H + hk) * p.d, *mine = sT + (STAGED ? wave * 32 * DP : 0);
    u32x4 fq[DP / 16];
    auto in_order = [&]() __attribute__((always_inline)) {           // what the wave's other lanes wrote is there (its LDS operations keep their order)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    // piece i of a lane: 16 bytes at (row, slot) of the tile
    auto row_at = [&](int i) __attribute__((always_inline)) { return (lane + 64 * i) / SL; };
    auto slot_of = [&](int i) __attribute__((always_inline)) { return (lane + 64 * i) % SL; };
    auto queries = [&](int t) __attribute__((always_inline)) {
        if constexpr (!STAGED) {
            load_q<DP>(p, row_of(p, b, hk, false, t * 32 + l31, rows), hi, fq);
        } else if (plain && t * 32 + 32 <= rows) {
            const char* at = reinterpret_cast<const char*>(q0 + t * 32 * p.q_n);
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                const int c = slot_of(i) * 8;
                fq[i] = *reinterpret_cast<const u32x4*>(at + (unsigned)(row_at(i) * (int)p.q_n + (c < p.d ? c : 0)) * 2u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                const Row row = row_of(p, b, hk, false, t * 32 + row_at(i), rows);
                const int c = slot_of(i) * 8;
                fq[i] = *reinterpret_cast<const u32x4*>(p.q + b * p.q_b + row.qi * p.q_n + row.h * p.q_h + (c < p.d ? c : 0));
            }
        }
    };
    auto settle = [&]() __attribute__((always_inline)) {
        if constexpr (STAGED) {
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) *reinterpret_cast<u32x4*>(mine + slot_at<DP>(row_at(i), slot_of(i))) = slot_of(i) * 8 < p.d ? fq[i] : u32x4{0u, 0u, 0u, 0u};
            in_order();
#pragma unroll
            for (int e = 0; e < DP / 16; ++e) fq[e] = read_row<DP>(mine, l31, e * 2 + hi);
            in_order();
        }
    };
    if (t0 < t1) queries(t0);
    const int len = p.lens ? max(0, min(p.lens[b], p.Nk)) : p.Nk, halves = max(1, (len + 15) / 16), blocks = (halves + 1) / 2;
    const u16 *kb = p.k + b * p.k_b + hk * p.k_h, *vb = p.v + b * p.v_b + hk * p.v_h;
    const unsigned char* mk = p.mask ? p.mask + b * p.mask_b : nullptr;
#pragma unroll
    for (int i = 0; i < NST; ++i) {
        const int id = tid + 256 * i, r = id / SL, slot = id % SL;
        if (r >= blocks * 32) break;                                  // (r grows with i)
        u32x4 rk = {0u, 0u, 0u, 0u}, rv = {0u, 0u, 0u, 0u};
        if (r < len && slot * 8 < p.d && (!mk || mk[r])) {
            rk = *reinterpret_cast<const u32x4*>(kb + r * p.k_n + slot * 8);
            rv = *reinterpret_cast<const u32x4*>(vb + r * p.v_n + slot * 8);
        }
        *reinterpret_cast<u32x4*>(sK + slot_at<DP>(r, slot)) = rk;
        *reinterpret_cast<u32x4*>(sV + slot_at<DP>(r, slot)) = rv;
    }
    const bool exists = tid < min(len, SHORT) && (!mk || mk[tid]);
    if (tid < SHORT) sE[tid] = exists ? 0.f : -INFINITY;
    if (!__syncthreads_or(exists)) {                                  // no key at all: zeros, whatever the queries hold
        for (int t = t0; t < t1; t += 4) {
            const Row row = row_of(p, b, hk, false, t * 32 + l31, rows);
            const long long id = ((long long)b * p.Nq + row.qi) * p.H + row.h;
#pragma unroll
            for (int n = 0; n < ND; ++n) store_row<BF>(p.o + id * p.d, zero16(), 0.f, n, hi, p.d, row.on);
            if (p.lse && hi == 0 && row.on) p.lse[((long long)b * p.H + row.h) * p.Nq + row.qi] = -INFINITY;
        }
        return;
    }
    if (t0 < t1) settle();
    auto walk = [&](auto which) __attribute__((always_inline)) {
        constexpr int NH = decltype(which)::value, NJ = (NH + 1) / 2; // half blocks of 16 keys, which an accumulator's first and last eight registers hold; blocks of 32
        for (int t = t0; t < t1; t += 4) {
            asm volatile("" ::: "memory");                            // keeps K and V in LDS: the compiler would carry them through the loop in registers, and spill
            f32x16 s[NJ];
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>(sE + j * 32 + 2 * r + 4 * hi);
#pragma unroll
                    for (int w = 0; w < 4; ++w) s[j][r + w] = x[w];
                }
#pragma unroll
                for (int e = 0; e < DP / 16; ++e) s[j] = mfma<BF>(read_row<DP>(sK, j * 32 + l31, e * 2 + hi), fq[e], s[j]);
            }
            if (t + 4 < t1) queries(t + 4);                           // the next tile's, into the registers that the scores have left
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 16 && 2 * j + (r >> 3) < NH; ++r) mx = fmaxf(mx, s[j][r]);
            const float m = half_max(mx) * p.c, ref = m == -INFINITY ? 0.f : m;
            float l = 0.f;
            f32x16 acc[ND];
#pragma unroll
            for (int n = 0; n < ND; ++n) acc[n] = zero16();
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                u32x4 fp[2];
#pragma unroll
                for (int r = 0; r < 16 && 2 * j + (r >> 3) < NH; r += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(fmaf(s[j][r], p.c, -ref)), p1 = __builtin_amdgcn_exp2f(fmaf(s[j][r + 1], p.c, -ref));
                    l += p0 + p1;
                    fp[r >> 3][(r >> 1) & 3] = pack2<BF>(p0, p1);
                }
#pragma unroll
                for (int e = 0; e < 2 && 2 * j + e < NH; ++e)
#pragma unroll
                    for (int n = 0; n < ND; ++n) acc[n] = mfma<BF>(read_tr<DP>(sV, j * 32 + e * 16, n * 32, lane), fp[e], acc[n]);
            }
            l = half_sum(l);
            const float inv = l > 0.f ? __builtin_amdgcn_rcpf(l) : 0.f;
            const Row row = row_of(p, b, hk, false, t * 32 + l31, rows);
            if (p.lse && hi == 0 && row.on) p.lse[((long long)b * p.H + row.h) * p.Nq + row.qi] = (m + __builtin_amdgcn_logf(l)) * LN2;
            if constexpr (!STAGED) {
                const long long id = ((long long)b * p.Nq + row.qi) * p.H + row.h;
#pragma unroll
                for (int n = 0; n < ND; ++n) store_row<BF>(p.o + id * p.d, acc[n], inv, n, hi, p.d, row.on);
            } else {
#pragma unroll
                for (int n = 0; n < ND; ++n)
#pragma unroll
                    for (int g = 0; g < 2; ++g) *reinterpret_cast<u32x4*>(mine + slot_at<DP>(l31, n * 4 + g * 2 + hi)) = eight<BF>(acc[n], inv, g);
                in_order();
                const bool whole = plain && t * 32 + 32 <= rows;
                char* at = reinterpret_cast<char*>(o0 + (long long)t * 32 * p.H * p.d);
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) {
                    const u32x4 x = read_row<DP>(mine, row_at(i), slot_of(i));
                    if (whole) {
                        if (slot_of(i) * 8 < p.d) *reinterpret_cast<u32x4*>(at + (unsigned)(row_at(i) * p.H * p.d + slot_of(i) * 8) * 2u) = x;
                    } else {
                        const Row to = row_of(p, b, hk, false, t * 32 + row_at(i), rows);
                        if (to.on && slot_of(i) * 8 < p.d) *reinterpret_cast<u32x4*>(p.o + (((long long)b * p.Nq + to.qi) * p.H + to.h) * p.d + slot_of(i) * 8) = x;
                    }
                }
                in_order();
            }
            if (t + 4 < t1) settle();
        }
    };
    switch (halves) {
        case 1: walk(Const<1>{}); break;
        case 2: walk(Const<2>{}); break;
        case 3: walk(Const<3>{}); break;
        case 4: walk(Const<4>{}); break;
        case 5: walk(Const<5>{}); break;
        default: walk(Const<6>{});
    }
}

// Joins the partial results of one row, a wave each: four groups of sixteen lanes take every fourth part, a lane eight channels
template <bool BF> __global__ void __launch_bounds__(256) k_ctx_join(const float* __restrict__ po, const float* __restrict__ pml, int parts, long long total, int d,
                                                                   int Nq, int H, u16* __restrict__ o, u16* __restrict__ o_lo, float* __restrict__ lse) {
    const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= total) return;
    const int lane = threadIdx.x & 63, grp = lane >> 4, c = (lane & 15) * 8;
    float m = -INFINITY;
    for (int s = lane; s < parts; s += 64) m = fmaxf(m, pml[(s * total + id) * 2]);
    m = wave_max_f32(m);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f, a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = grp; s < parts; s += 4) {
        const f32x2 x = *reinterpret_cast<const f32x2*>(pml + (s * total + id) * 2);
        const float f = __builtin_amdgcn_exp2f(x[0] - ref);          // a part without a key: exp2(-inf) = 0
        const float* t = po + (s * total + id) * d + (c < d ? c : 0);
        const f32x4 t0 = *reinterpret_cast<const f32x4*>(t), t1 = *reinterpret_cast<const f32x4*>(t + 4);
        l += f * x[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            a[e] += f * t0[e];
            a[e + 4] += f * t1[e];
        }
    }
#pragma unroll
    for (int w = 16; w < 64; w *= 2) {
        l += __shfl_xor(l, w, 64);
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] += __shfl_xor(a[e], w, 64);
    }
    if (grp) return;
    const float inv = l > 0.f ? __builtin_amdgcn_rcpf(l) : 0.f;
    if (c < d) {
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] *= inv;
        *reinterpret_cast<u32x4*>(o + id * d + c) = u32x4{pack2<BF>(a[0], a[1]), pack2<BF>(a[2], a[3]), pack2<BF>(a[4], a[5]), pack2<BF>(a[6], a[7])};
        if (o_lo) *reinterpret_cast<u32x4*>(o_lo + id * d + c) = u32x4{left2<BF>(a[0], a[1]), left2<BF>(a[2], a[3]), left2<BF>(a[4], a[5]), left2<BF>(a[6], a[7])};
    }
    if (lse && c == 0) {
        const long long bq = id / H;
        lse[((bq / Nq) * H + id % H) * Nq + bq % Nq] = (m + __builtin_amdgcn_logf(l)) * LN2;
    }
}

// How a call is laid out: which rows a block owns, how the keys are dealt out, which launches that takes
struct Plan {
    bool one_pass;             // k_ctx_short
    int mode, chunks, per_chunk;
    Deal first, second;
    int parts;                 // partial results to join (0: the kernel writes the result)
};
// `tiles` tiles of work in each of `blocks` places: how many of them a block takes.  Where the places alone leave part of the chip idle the tiles are dealt
// out in runs: as many as make the rounds that `slots` resident blocks take shortest (a block's start and its partial results count as two tiles), at least `least` tiles each
// (2 x 1000 rows x 4000 keys, 10 heads of 128: 3 runs, 480 blocks, 65 us; 4 runs, 640 blocks in two rounds, 77 us).  From 384 places on nothing is dealt out: dealt / as it
// is, fp16, 4 x 1456 rows x 2311 keys: 8 heads of 64 (384 places) 60 / 52 us, of 128 104 / 79; 10 heads (480) 78 / 55 and 87 / 87; 12 heads (576) 91 / 70 and
// 150 / 140.  Below: 2 x 1000 x 4000, 10 heads (160) 50 / 71 and 68 / 106; 2 x 1900 x 4000, 10 heads (300) 76 / 88 and 124 / 128; but 3 x 1900 x 2000, 8 heads
// (360), 57 / 46 and 93 / 69; and single tokens would gain above: 8 x 1 x 20000, 80 heads (640) 553 / 739 and 1092 / 1187.
long long dealt(long long blocks, long long tiles, long long slots, long long least) {
    long long best = tiles, cost = (blocks + slots - 1) / slots * (tiles + 2);
    for (int r = 1; blocks < 384 && r <= 8; ++r) {                    // as many runs as r rounds hold
        long long c = r * slots / blocks;
        if (c > tiles / least) c = tiles / least;
        if (c < 2) continue;
        const long long per = (tiles + c - 1) / c, rounds = (blocks * ((tiles + per - 1) / per) + slots - 1) / slots;
        if (rounds * (per + 2) < cost) {
            cost = rounds * (per + 2);
            best = per;
        }
    }
    return best < 1 ? 1 : best;
}
Plan make_plan(int B, int Nq, int Np, int Nk, int H, int Hk, int d, bool short_ok) {
    Plan s{};
    const int G = H / Hk;
    const long long rows = (long long)Nq * G, heads = (long long)B * Hk;
    const int slots = d <= 64 ? 768 : 512;                            // blocks that the chip holds: three a CU, or two
    if (Np == 0 && Nk <= SHORT && rows >= 64 && short_ok) {            // (k_ctx_short has no limit by row, and writes no o_lo)
        // (k_ctx_short / k_ctx_attn: 28 x 4096 rows, 5 heads of 64, 33 keys 31 / 44 us, 77 keys 36 to 41 / 58, 96 keys 40 / 55; 14 x 4096, 8 heads, 77 keys of 96
        // 42 / 68, of 128 73 / 79; 256 x 64 rows, 16 heads of 64 39 / 47.  With room for 128 keys, 120 of them: of 64 51 / 54, of 96 76 / 75, of 128 94 / 82;
        // 28 x 1024 rows, 10 heads of 64 28.6 / 27.6)
        // the keys are staged once a block: one round of the blocks that the chip holds, or, from half of that in heads alone, rounds of
        // blocks small enough for the last one to weigh little; at least two tiles a wave
        // (14 x 4096 rows x 77 keys, 8 heads of 96: 448 blocks 42 us, 672 in two rounds 51)
        const long long tiles = (rows + 31) / 32, want = heads <= slots / 2 ? slots / heads : (4 * slots + heads - 1) / heads;
        const long long per = (tiles + want - 1) / want;
        s.one_pass = true;
        s.per_chunk = (int)(per < 8 ? 8 : (per + 3) / 4 * 4);
        s.chunks = (int)((tiles + s.per_chunk - 1) / s.per_chunk);
        return s;
    }
    auto deal = [](Deal& w, long long places, int key_tiles, int slots) {      // at least 4 tiles (256 or 512 keys): below, a joining launch costs more than it spreads
        const long long per = dealt(places, key_tiles, slots, 4);
        w.splits = key_tiles > per ? (int)((key_tiles + per - 1) / per) : 1;
        w.per_split = (int)per;
        w.blocks = (int)(places * w.splits);
    };
    // Few rows: where a wave's 32 columns hold all rows of a key head the keys are what has to be read, and k_ctx_attn's few_rows reads them faster
    // (64 samples of 16 rows over 2000 keys, 16 heads of 64: 111 us, 4.7 TB/s, for 124 as many_rows; 256 samples over 77 keys 33 us for 51).
    // Stacked: a row tile of one sample alone would be mostly empty, so the rows of all samples share row tiles for the prefix, where what that saves
    // pays for the joining launch (single tokens, stacked / each sample by itself: 64 samples over 1024 prefix keys 42.8 / 48.1 us, over 512 38.4 / 37.0;
    // 4 over 16384 23.7 / 48.2, over 512 23.5 / 19.8; 1024 over 64 59.4 / 63.2).  2^26 rows are what the joining launch takes.
    const bool few = rows <= 32, stack = B > 1 && rows < 128 && (long long)B * Np >= 32768 && rows * heads < (1ll << 26);
    const bool stack_few = few && rows * B <= 32;
    s.mode = !few ? MANY : (!stack || stack_few) ? FEW : MIXED;
    if (stack) {
        const int kt = stack_few ? 128 : 64;
        s.first.stacked = 1;
        s.first.np = Np;
        s.first.xtiles = stack_few ? 1 : (int)((rows * B + 127) / 128);
        deal(s.first, (long long)Hk * s.first.xtiles, (Np + kt - 1) / kt, slots);
        s.parts = s.first.splits;
    }
    if (Nk > 0 || !stack) {
        const int kt = few ? 128 : 64;
        s.second.np = stack ? 0 : Np;
        s.second.xtiles = few ? 1 : (int)((rows + 127) / 128);
        s.second.part0 = s.parts;
        deal(s.second, heads * s.second.xtiles, (Nk + kt - 1) / kt + (s.second.np + kt - 1) / kt, slots);
        s.parts += s.second.splits;
    }
    if (s.parts == 1) s.parts = 0;
    return s;
}

template <bool BF, int DP> void launch_fwd(const AttnArgs& p, const Plan& s, hipStream_t st) {
    if (s.one_pass) {
        const dim3 grid((unsigned)((long long)s.chunks * p.B * p.Hk));
        hipLaunchKernelGGL((k_ctx_short<BF, DP>), grid, dim3(256), 0, st, p, s.chunks, s.per_chunk);
        return;
    }
    const dim3 grid((unsigned)(s.first.blocks + s.second.blocks));
    if (s.mode == MANY) hipLaunchKernelGGL((k_ctx_attn<BF, DP, MANY>), grid, dim3(256), 0, st, p, s.first, s.second);
    else if (s.mode == FEW) hipLaunchKernelGGL((k_ctx_attn<BF, DP, FEW>), grid, dim3(256), 0, st, p, s.first, s.second);
    else hipLaunchKernelGGL((k_ctx_attn<BF, DP, MIXED>), grid, dim3(256), 0, st, p, s.first, s.second);
    if (s.parts) {
        const long long total = (long long)p.B * p.Nq * p.H;
        hipLaunchKernelGGL((k_ctx_join<BF>), dim3((unsigned)((total + 3) / 4)), dim3(256), 0, st, p.po, p.pml, s.parts, total, p.d, p.Nq, p.H, p.o, p.o_lo, p.lse);
    }
}

// ------------------------------------------------------------------------------------------------------------------------------------
// Backward.  With L = lse log2 e and D = sum_keys p dp of a row:  p = exp2(s c - L),  dp = do v^T,  ds = p (dp - D),
//   dv = p^T do,   dk = scale ds^T q,   dq = scale ds k.
// p and ds are rounded once to the storage type before they enter a product.  fp16 needs both kept away from its subnormals (p of a row over
// 4096 keys is 2^-12, its ds smaller still): p is carried as 2^12 p, and dp - D with a power of two that brings the largest in sight to 1..4, so ds
// stays below 2^14 and a subnormal's half step is 2^-37 of the largest |dp - D| -- exact factors that leave in fp32 at the end; accumulators are
// rescaled where the power changes.
struct BwdArgs {
    const u16 *q, *k, *v, *o, *o_lo, *go;
    long long q_b, q_n, q_h, k_b, k_n, k_h, v_b, v_n, v_h, g_b, g_n, g_h;
    const float* lse;
    float* delta;              // [B][H][Nq]: D, written by the dq kernel for the dk / dv kernel
    const int* lens;
    const unsigned char* mask;
    long long mask_b;
    u16 *dq, *dk, *dv;         // contiguous [B][Nq][H][d], [Bk][Nk][Hk][d]
    float* part;               // [chunks][2][Bk][Nk][Hk][d] or null: one chunk, written as it is
    int B, Bk, Nq, Nk, H, Hk, G, d;
    float c, scale;
    int xtiles, chunks, per_chunk;
};

constexpr float P_LOG2 = 12.f, P_BACK = 2.44140625e-4f;                         // fp16: p as 2^12 p
// 2^-floor(log2 m), at most 2^60
__device__ __forceinline__ float power_for(float m) { return __uint_as_float((254u - max(67u, min(__float_as_uint(m) >> 23, 253u))) << 23); }

// dq: a wave owns 32 rows as accumulator columns, the block's waves share key tiles of 64 (the forward kernel's arrangement); K serves as rows (scores)
// and transposed (ds k).  Three products: 2 x 16 heads x 4096 x 4096 of 128 (bf16) 377 us, 1090 TFLOP/s; 4 x 10 heads x 1456 x 2311 of 64 (fp16) 84 us, 620
// (480 blocks: two on most CUs where three would fit).  D comes out of the saved result: o was rounded, o_lo holds what the rounding left.
template <bool BF, int DP> __global__ void __launch_bounds__(256, DP == 64 ? 3 : 2) k_ctx_bwd_q(BwdArgs p) {
    constexpr int KT = 64, ND = DP / 32, TILE = KT * DP;
    __shared__ __attribute__((aligned(16))) u16 sK[2 * TILE], sV[2 * TILE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, hi = lane >> 5;
    int y, xt;
    block_of(p.xtiles, y, xt);
    const int hk = y % p.Hk, b = y / p.Hk, rows = p.Nq * p.G;
    const int len = p.lens ? max(0, min(p.lens[b], p.Nk)) : p.Nk, T = (len + KT - 1) / KT;
    const u16 *kb = p.k + b * p.k_b + hk * p.k_h, *vb = p.v + b * p.v_b + hk * p.v_h;
    const unsigned char* mk = p.mask ? p.mask + b * p.mask_b : nullptr;
    Fetch<DP> fk, fv;
    fk.init(tid, p.k_n, p.d);
    fv.init(tid, p.v_n, p.d);
    unsigned long long live = 0;
    auto fetch = [&](int t, int buf) __attribute__((always_inline)) {
        const int k0 = t * KT, n = len - k0;
        live = n >= KT ? ~0ull : (1ull << n) - 1;
        if (mk) live = __ballot(lane < n && mk[k0 + min(lane, n - 1)]);
        fk.tile(kb + k0 * p.k_n, p.k_n, live, sK + buf * TILE, tid, wave);
        fv.tile(vb + k0 * p.v_n, p.v_n, live, sV + buf * TILE, tid, wave);
    };
    if (T > 0) fetch(0, 0);
    const int r = xt * 128 + wave * 32 + l31;
    const bool on = r < rows;
    const int rr = min(r, rows - 1), qi = rr / p.G, h = hk * p.G + rr % p.G;
    const long long id = ((long long)b * p.Nq + qi) * p.H + h;
    u32x4 fq[DP / 16], fg[DP / 16];
    float D = 0.f;
    const long long bhq = ((long long)b * p.H + h) * p.Nq + qi;
    const float lse = p.lse[bhq];
    const bool none = lse == -INFINITY;                                         // a row without a key is taken as zeros, whatever it holds: p = 0 would be multiplied by it
    {
        const u16 *qp = p.q + b * p.q_b + qi * p.q_n + h * p.q_h, *gp = p.go + b * p.g_b + qi * p.g_n + h * p.g_h;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            const int at = s * 16 + hi * 8, a = at < p.d ? at : 0;
            fq[s] = *reinterpret_cast<const u32x4*>(qp + a);
            fg[s] = *reinterpret_cast<const u32x4*>(gp + a);
            const u32x4 fo = *reinterpret_cast<const u32x4*>(p.o + id * p.d + a), fl = *reinterpret_cast<const u32x4*>(p.o_lo + id * p.d + a);
            if (at >= p.d || none) fq[s] = fg[s] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
            for (int e = 0; e < 4; ++e) D = dot2<BF>(fg[s][e], fl[e], dot2<BF>(fg[s][e], fo[e], D));
        }
    }
    D = half_sum(D);
    const float L = none ? INFINITY : lse * LOG2E - (BF ? 0.f : P_LOG2);         // (p = 0)
    if (on && hi == 0) p.delta[bhq] = D;
    float power = BF ? 1.f : 1.152921504606846976e18f;                          // this row's factor of ds
    f32x16 acc[ND];
#pragma unroll
    for (int n = 0; n < ND; ++n) acc[n] = zero16();
    landed();
    auto work = [&](auto which, int t) __attribute__((always_inline)) {
        constexpr int buf = decltype(which)::value;
        const unsigned long long now = live;
        if (t + 1 < T) fetch(t + 1, buf ^ 1);
        auto half = [&](auto which_half) __attribute__((always_inline)) {
            constexpr int j = decltype(which_half)::value;
            f32x16 s, z;
#pragma unroll
            for (int e = 0; e < DP / 16; ++e) s = mfma<BF>(read_row<DP>(sK + buf * TILE, j * 32 + l31, e * 2 + hi), fq[e], e ? s : zero16());
#pragma unroll
            for (int e = 0; e < DP / 16; ++e) z = mfma<BF>(read_row<DP>(sV + buf * TILE, j * 32 + l31, e * 2 + hi), fg[e], e ? z : zero16());
            if (now != ~0ull) hide(s, (unsigned)(now >> (32 * j)), 1 << 30, hi);
#pragma unroll
            for (int e = 0; e < 16; ++e) z[e] -= D;
            if (!BF) {
                float m = fabsf(z[0]);
#pragma unroll
                for (int e = 1; e < 16; ++e) m = fmaxf(m, fabsf(z[e]));
                if (__builtin_expect(__any(m * power > 4.f), 0)) {
                    const float f = fminf(power, power_for(half_max(m)));      // both lane halves hold the same row
#pragma unroll
                    for (int n = 0; n < ND; ++n)
#pragma unroll
                        for (int e = 0; e < 16; ++e) acc[n][e] *= f / power;
                    power = f;
                }
            }
            u32x4 fd[2];
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                float x = __builtin_amdgcn_exp2f(fmaf(s[e], p.c, -L)) * z[e], w = __builtin_amdgcn_exp2f(fmaf(s[e + 1], p.c, -L)) * z[e + 1];
                if (!BF) {
                    x *= power;
                    w *= power;
                }
                fd[e >> 3][(e >> 1) & 3] = pack2<BF>(x, w);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int n = 0; n < ND; ++n) acc[n] = mfma<BF>(read_tr<DP>(sK + buf * TILE, j * 32 + e * 16, n * 32, lane), fd[e], acc[n]);
        };
        half(Const<0>{});
        half(Const<1>{});
        landed();
    };
    for (int t = 0; t < T; t += 2) {
        work(Const<0>{}, t);
        if (t + 1 < T) work(Const<1>{}, t + 1);
    }
    const float back = p.scale / power * (BF ? 1.f : P_BACK);
#pragma unroll
    for (int n = 0; n < ND; ++n) store_row<BF>(p.dq + id * p.d, acc[n], back, n, hi, p.d, on);
}

// The 32 lanes of a half hold 32 keys of 16 rows (registers): the rows' sums over the lanes.  Registers are folded pairwise across 16-lane groups first, then
// summed within them; lane i < 8 of a group ends with the sum of row register 2 i (+ 1 in the upper group).
__device__ __forceinline__ float rows_sum(const f32x16& x, int lane) {
    float a[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const auto w = __builtin_amdgcn_permlane16_swap(__float_as_uint(x[2 * i]), __float_as_uint(x[2 * i + 1]), false, false);
        a[i] = __uint_as_float(w[0]) + __uint_as_float(w[1]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        a[i] += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(a[i]), 0x128, 0xf, 0xf, true));     // row_ror:8
        a[i] += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(a[i]), 0x124, 0xf, 0xf, true));     // row_ror:4
        a[i] += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(a[i]), 0x122, 0xf, 0xf, true));     // row_ror:2
        a[i] += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(a[i]), 0x121, 0xf, 0xf, true));     // row_ror:1
    }
    float v = a[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) v = (lane & 7) == i ? a[i] : v;
    return v;
}

// dk and dv: a wave owns 32 keys as accumulator columns (K, V in registers), the block 128, and walks over tiles of 64 queries of one head: the heads of the
// group, and the samples where they share one context, one after the other.  FUSED (at most 128 keys): the block holds every key of its rows, so D is summed
// here from the unrounded p dp (four partial sums a row through LDS) and dq comes out of the same pass -- ds goes through LDS once more, each wave takes
// its share of the [64][d] tile of ds k -- and q and do are all that is read per row.
// DV, DK: which of the two the block accumulates.  SHARED: whether not FUSED blocks walk over the samples of one context; a variant of its own, for what that
// asks at each sample makes the compiler lay out the other's loop worse (4 x 10 heads x 1456 x 2311 of 64, fp16, nothing shared: 125 us as one variant, 105 as two).
// FUSED 28 x 4096 rows x 77 keys, 5 heads of 64, forward and gradients: 171 us bf16, as three passes 234; 14 x 4096, 8 heads of 128: 295 and 375; with 120 keys 185 / 239
// and 306 / 388.  77 keys take no less than 96 would: a wave owns 32 keys, so the fourth wave has none, and the third 13.
// Not FUSED, 4 x 10 heads x 1456 x 2311 of 64 (fp16): 116 us, 595 TFLOP/s; 2 x 16 heads on 4 x 4096 x 4096 of 128 (bf16): 833 us, 660.
template <int DP, bool FUSED> struct BwdLds {
    __attribute__((aligned(16))) u16 q[2 * 64 * DP], g[2 * 64 * DP], k[FUSED ? 128 * DP : 8], s[FUSED ? 128 * 64 : 8];
    __attribute__((aligned(16))) float l[2][64], d[FUSED ? 4 : 2][64], m[4];
};
template <bool BF, int DP, bool FUSED, bool DV, bool DK, bool SHARED> __device__ __forceinline__ void keys_walk(const BwdArgs& p, int y, int kt, BwdLds<DP, FUSED>& lds) {
    constexpr int RT = 64, ND = DP / 32, TILE = RT * DP;
    u16 *sQ = lds.q, *sG = lds.g, *sK = lds.k, *sS = lds.s;
    float(*sL)[64] = lds.l;
    float(*sD)[64] = lds.d;
    float* sM = lds.m;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, hi = lane >> 5;
    const int chunk = y % p.chunks;
    y /= p.chunks;
    const int hk = y % p.Hk, bk = y / p.Hk;                                      // bk: sample of k and v
    const bool shared = FUSED ? p.Bk < p.B : SHARED;
    const int tiles = (p.Nq + RT - 1) / RT;                                      // of one head
    const long long all = (long long)tiles * p.G * (shared ? p.B : 1), t0 = (long long)chunk * p.per_chunk;
    int count = (int)((t0 + p.per_chunk < all ? t0 + p.per_chunk : all) - t0);
    const int key = kt * 128 + wave * 32 + l31;
    const bool in = key < p.Nk;
    // a key that no sample of this block has is taken as zero, so nothing that lies there reaches a product
    auto exists = [&](int k, int b) __attribute__((always_inline)) { return k < p.Nk && (!p.lens || k < p.lens[b]) && (!p.mask || p.mask[b * p.mask_b + k]); };
    auto lives = [&](int b) __attribute__((always_inline)) { return exists(key, b); };
    bool any = false;
    if (shared) {
        for (int i = 0; i < p.B; ++i) any |= lives(i);
    } else {
        any = lives(bk);
    }
    if (!FUSED && !__syncthreads_or(any)) count = 0;                             // all 128 keys are dead: their gradients are zero
    struct At {                                                                  // a tile: sample, head of the group, first query
        int b, g, i;
    };
    auto step = [&](At& x) __attribute__((always_inline)) {
        if (++x.i == tiles) {
            x.i = 0;
            if (++x.g == p.G) {
                x.g = 0;
                ++x.b;
            }
        }
    };
    At now;
    now.i = (int)(t0 % tiles);
    now.g = (int)(t0 / tiles % p.G);
    now.b = shared ? (int)(t0 / tiles / p.G) : bk;
    At next = now;                                                               // the tile to be fetched next
    Fetch<DP> fq, fg;
    fq.init(tid, p.q_n, p.d);
    fg.init(tid, p.g_n, p.d);
    float rL = INFINITY, rD = 0.f;
    // A sample that has none of the block's keys adds nothing to their gradients; its rows are taken as zeros, for its probabilities of zero would still be
    // multiplied by what they hold, and a padded sample's rows may hold NaN.  (Not FUSED, one sample's own keys: such a block has no tiles.)
    int asked = -1, have = p.Nq;                                                 // the sample of the next fetch, its rows that are fetched
    auto ask = [&](int b) __attribute__((always_inline)) {                       // (every wave looks at the block's 128 keys)
        if (b == asked || b >= p.B) return;
        asked = b;
        if (p.lens || p.mask) have = __builtin_amdgcn_readfirstlane(__any(exists(kt * 128 + lane, asked) || exists(kt * 128 + 64 + lane, asked)) ? p.Nq : 0);
    };
    auto fetch = [&](int buf) __attribute__((always_inline)) {
        const int q0 = next.i * RT, n = max(0, have - q0), h = hk * p.G + next.g;
        const unsigned long long live = n >= RT ? ~0ull : (1ull << n) - 1;
        fq.tile(p.q + next.b * p.q_b + h * p.q_h + q0 * p.q_n, p.q_n, live, sQ + buf * TILE, tid, wave);
        fg.tile(p.go + next.b * p.g_b + h * p.g_h + q0 * p.g_n, p.g_n, live, sG + buf * TILE, tid, wave);
        if (tid < RT) {
            const long long at = ((long long)next.b * p.H + h) * p.Nq + min(q0 + tid, p.Nq - 1);
            const float lse = p.lse[at];
            rL = tid >= n || lse == -INFINITY ? INFINITY : lse * LOG2E - (BF ? 0.f : P_LOG2);
            if (!FUSED) rD = tid < n ? p.delta[at] : 0.f;
        }
        step(next);
    };
    auto settle = [&](int buf) __attribute__((always_inline)) {
        if (tid < RT) {
            sL[buf][tid] = rL;
            if (!FUSED) sD[buf][tid] = rD;
        }
    };
    if (count > 0) fetch(0);
    u32x4 fk[DP / 16], fv[DP / 16];
    {
        const int kk = in ? key : 0;
        const u16 *kp = p.k + bk * p.k_b + kk * p.k_n + hk * p.k_h, *vp = p.v + bk * p.v_b + kk * p.v_n + hk * p.v_h;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            const int at = s * 16 + hi * 8, a = at < p.d ? at : 0;
            fk[s] = *reinterpret_cast<const u32x4*>(kp + a);
            if (DK) fv[s] = *reinterpret_cast<const u32x4*>(vp + a);
            if (at >= p.d || !any) fk[s] = fv[s] = u32x4{0u, 0u, 0u, 0u};
        }
    }
    if (FUSED || shared) {                                                       // the first tile is on its way already: fetched anew in the rare case
        ask(now.b);
        if (!have && count > 0) {
            landed();
            next = now;
            fetch(0);
        }
        if (shared) ask(next.b);
    }
    bool live = shared ? lives(now.b) : any;
    // FUSED: K for dq, zero where the rows' sample has no such key (another sample of a shared context may, with anything in it)
    auto keep_k = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) *reinterpret_cast<u32x4*>(sK + slot_at<DP>(wave * 32 + l31, s * 2 + hi)) = live ? fk[s] : u32x4{0u, 0u, 0u, 0u};
    };
    if constexpr (FUSED) keep_k();
    bool whole = (!FUSED && !shared) || __all(live);                             // one sample's own keys, not FUSED: a dead key spoils its own column alone, which is not stored
    f32x16 ak[ND], av[ND];
#pragma unroll
    for (int n = 0; n < ND; ++n) ak[n] = av[n] = zero16();
    float power = BF ? 1.f : 1.152921504606846976e18f;                          // factor of ds in ak: of this key's column, FUSED: of the block
    settle(0);
    landed();

    // s -> p (fp32), z = dp; the tile's rows i * 32 ..
    auto scores = [&](int buf, int i, f32x16& s, f32x16& z) __attribute__((always_inline)) {
        const u16 *tq = sQ + buf * TILE, *tg = sG + buf * TILE;
#pragma unroll
        for (int e = 0; e < DP / 16; ++e) s = mfma<BF>(read_row<DP>(tq, i * 32 + l31, e * 2 + hi), fk[e], e ? s : zero16());
        if (DK)
#pragma unroll
            for (int e = 0; e < DP / 16; ++e) z = mfma<BF>(read_row<DP>(tg, i * 32 + l31, e * 2 + hi), fv[e], e ? z : zero16());
        if (!whole)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (!live) {
                    s[e] = -INFINITY;
                    if (FUSED) z[e] = 0.f;                                        // D sums over the keys: 0 times what lies there may be NaN
                }
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const f32x4 L = *reinterpret_cast<const f32x4*>(&sL[buf][i * 32 + 2 * e + 4 * hi]);
#pragma unroll
            for (int w = 0; w < 4; ++w) s[e + w] = __builtin_amdgcn_exp2f(fmaf(s[e + w], p.c, -L[w]));
        }
    };
    auto pack = [&](const f32x16& x, float f, u32x4 (&o)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 16; e += 2) o[e >> 3][(e >> 1) & 3] = pack2<BF>(x[e] * f, x[e + 1] * f);
    };
    auto products = [&](int buf, int i, const u32x4 (&fp)[2], const u32x4 (&fd)[2]) __attribute__((always_inline)) {
        const u16 *tq = sQ + buf * TILE, *tg = sG + buf * TILE;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int n = 0; n < ND; ++n) {
                if (DV) av[n] = mfma<BF>(read_tr<DP>(tg, i * 32 + e * 16, n * 32, lane), fp[e], av[n]);
                if (DK) ak[n] = mfma<BF>(read_tr<DP>(tq, i * 32 + e * 16, n * 32, lane), fd[e], ak[n]);
            }
    };
    auto move_power = [&](float f) __attribute__((always_inline)) {
        const float by = f / power;
#pragma unroll
        for (int n = 0; n < ND; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) ak[n][e] *= by;
        power = f;
    };
    for (int t = 0; t < count; ++t) {
        const int buf = t & 1;
        const bool more = t + 1 < count;
        if (more) fetch(buf ^ 1);
        if constexpr (!FUSED) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                f32x16 s, z;
                scores(buf, i, s, z);
                u32x4 fp[2], fd[2];
                if (DV) pack(s, 1.f, fp);
                if (DK) {
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const f32x4 D = *reinterpret_cast<const f32x4*>(&sD[buf][i * 32 + 2 * e + 4 * hi]);
#pragma unroll
                        for (int w = 0; w < 4; ++w) z[e + w] -= D[w];
                    }
                    if (!BF) {
                        float m = fabsf(z[0]);
#pragma unroll
                        for (int e = 1; e < 16; ++e) m = fmaxf(m, fabsf(z[e]));
                        if (__builtin_expect(__any(m * power > 4.f), 0)) move_power(fminf(power, power_for(half_max(m))));
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) z[e] *= s[e];
                    pack(z, BF ? 1.f : power, fd);
                }
                products(buf, i, fp, fd);
            }
            if (more) settle(buf ^ 1);
            landed();
        } else {
            f32x16 s[2], z[2];
            // D: this wave's keys' share of each row, p in its own scale
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                scores(buf, i, s[i], z[i]);
                f32x16 x;
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = s[i][e] * z[i][e];
                const float sum = rows_sum(x, lane) * (BF ? 1.f : P_BACK);
                const int e = 2 * (lane & 7) + ((lane >> 4) & 1);
                if ((lane & 15) < 8) sD[wave][i * 32 + (e & 3) + 8 * (e >> 2) + 4 * hi] = sum;
            }
            if (!BF) {
                float m = 0.f;
#pragma unroll
                for (int e = 0; e < 16; ++e) m = fmaxf(fmaxf(m, fabsf(z[0][e])), fabsf(z[1][e]));
                m = wave_max_f32(m);
                if (lane == 0) sM[wave] = m;
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");    // (the next tile's fetch stays under way)
            if (!BF) {
                const float m = fmaxf(fmaxf(sM[0], sM[1]), fmaxf(sM[2], sM[3]));  // |dp - D| <= 2 m
                if (m > 0.f && power_for(m) != power) move_power(power_for(m));
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                u32x4 fp[2], fd[2];
                pack(s[i], 1.f, fp);
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    f32x4 D = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        const f32x4 w = *reinterpret_cast<const f32x4*>(&sD[v][i * 32 + 2 * e + 4 * hi]);
#pragma unroll
                        for (int u = 0; u < 4; ++u) D[u] += w[u];
                    }
#pragma unroll
                    for (int w = 0; w < 4; ++w) z[i][e + w] = (z[i][e + w] - D[w]) * s[i][e + w];
                }
                pack(z[i], BF ? 1.f : power, fd);
#pragma unroll
                for (int e = 0; e < 16; e += 4)                                 // [key][row]: rows i 32 + 2 e + 4 hi + 0..3
                    *reinterpret_cast<u32x2*>(sS + slot_at<RT>(wave * 32 + l31, i * 4 + (e >> 2)) + 4 * hi) = u32x2{fd[e >> 3][(e >> 1) & 3], fd[e >> 3][((e >> 1) & 3) + 1]};
                products(buf, i, fp, fd);
            }
            if (more) settle(buf ^ 1);
            landed();
            const float to_dq = p.scale / power * (BF ? 1.f : P_BACK);
            const int h = hk * p.G + now.g;
            for (int w = wave; w < 2 * ND; w += 4) {
                const int i = w & 1, n = w >> 1;
                f32x16 acc = zero16();
#pragma unroll
                for (int e = 0; e < 8; ++e) acc = mfma<BF>(read_tr<DP>(sK, e * 16, n * 32, lane), read_tr<RT>(sS, e * 16, i * 32, lane), acc);
                const int qi = now.i * RT + i * 32 + l31;
                const long long id = ((long long)now.b * p.Nq + min(qi, p.Nq - 1)) * p.H + h;
                store_row<BF>(p.dq + id * p.d, acc, to_dq, n, hi, p.d, qi < p.Nq);
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");    // sS and sD are written again in the next round
        }
        const int b = now.b;
        step(now);
        if (shared && more) {
            ask(next.b);
            if (now.b != b) {
                live = lives(now.b);
                whole = __all(live);
                if constexpr (FUSED) keep_k();                                    // (every wave has read the old rows, and reads the new ones two barriers on)
            }
        }
    }
    const float to_k = any ? p.scale / power * (BF ? 1.f : P_BACK) : 0.f, to_v = any ? (BF ? 1.f : P_BACK) : 0.f;
    if (!any)
#pragma unroll
        for (int n = 0; n < ND; ++n) ak[n] = av[n] = zero16();                   // (they may hold infinities)
    const long long at = (((long long)bk * p.Nk + (in ? key : 0)) * p.Hk + hk) * p.d, plane = (long long)p.Bk * p.Nk * p.Hk * p.d;
#pragma unroll
    for (int n = 0; n < ND; ++n) {
        if (!p.part) {
            if (DK) store_row<BF>(p.dk + at, ak[n], to_k, n, hi, p.d, in);
            if (DV) store_row<BF>(p.dv + at, av[n], to_v, n, hi, p.d, in);
        } else if (in) {
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int c = n * 32 + 2 * e + 4 * hi;
                if (c >= p.d) continue;
                float* o = p.part + 2 * chunk * plane + at + c;
                if (DK) *reinterpret_cast<f32x4*>(o) = f32x4{ak[n][e] * to_k, ak[n][e + 1] * to_k, ak[n][e + 2] * to_k, ak[n][e + 3] * to_k};
                if (DV) *reinterpret_cast<f32x4*>(o + plane) = f32x4{av[n][e] * to_v, av[n][e + 1] * to_v, av[n][e + 2] * to_v, av[n][e + 3] * to_v};
            }
        }
    }
}

// Wide heads, not FUSED: the accumulators of both gradients and K, V leave room for one wave a SIMD only, which waits more than it works; so half of the
// blocks take dk and the other half dv (five products for four, at two waves a SIMD).  Forward and gradients, separate / together: 4 x 10 heads x 1456 x 2311
// of 96 fp16 357 / 363 us, bf16 327 / 371, of 128 fp16 444 / 461, bf16 420 / 421; 2 x 16 heads on 4 x 4096 x 4096 of 96 fp16 1192 / 1214, bf16 1102 / 1269, of 128 fp16
// 1521 / 1590, bf16 1429 / 1441.
template <bool BF, int DP, bool FUSED, bool SHARED = false> __global__ void __launch_bounds__(256, DP == 64 || !FUSED ? 2 : 1) k_ctx_bwd_kv(BwdArgs p) {
    __shared__ BwdLds<DP, FUSED> lds;
    int y, kt;
    block_of(p.xtiles, y, kt);
    if constexpr (FUSED || DP == 64) {
        keys_walk<BF, DP, FUSED, true, true, SHARED>(p, y, kt, lds);
    } else {
        if (kt & 1) keys_walk<BF, DP, FUSED, true, false, SHARED>(p, y, kt >> 1, lds);
        else keys_walk<BF, DP, FUSED, false, true, SHARED>(p, y, kt >> 1, lds);
    }
}

// dk (y = 0) and dv (y = 1): the chunks' partial sums in their order
template <bool BF> __global__ void __launch_bounds__(256) k_ctx_bwd_sum(const float* __restrict__ part, int chunks, long long plane, u16* __restrict__ dk, u16* __restrict__ dv) {
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= plane) return;
    const float* o = part + blockIdx.y * plane + i;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int c = 0; c < chunks; ++c) {
        const f32x4 t = *reinterpret_cast<const f32x4*>(o + 2 * c * plane);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] += t[e];
    }
    *reinterpret_cast<u32x2*>((blockIdx.y ? dv : dk) + i) = u32x2{pack2<BF>(a[0], a[1]), pack2<BF>(a[2], a[3])};
}

struct BwdPlan {
    bool fused;
    int ktiles, chunks, per_chunk;
    long long delta_floats, part_floats;
};
BwdPlan make_bwd_plan(int B, int Bk, int Nq, int Nk, int H, int Hk, int d) {
    BwdPlan s{};
    s.fused = Nk <= 128;
    s.ktiles = (Nk + 127) / 128;
    const long long tiles = ((long long)Nq + 63) / 64 * (H / Hk) * (Bk < B ? B : 1), blocks = (long long)Bk * Hk * s.ktiles;
    const long long best = dealt(blocks, tiles, s.fused && d > 64 ? 256 : 512, 2);
    s.per_chunk = (int)best;
    s.chunks = (int)((tiles + best - 1) / best);
    s.delta_floats = s.fused ? 0 : ((long long)B * H * Nq + 3) / 4 * 4;
    s.part_floats = s.chunks > 1 ? 2ll * s.chunks * Bk * Nk * Hk * d : 0;
    return s;
}

template <bool BF, int DP> void launch_bwd(BwdArgs p, const BwdPlan& s, bool want_kv, hipStream_t st) {
    const unsigned kv_blocks = (unsigned)(s.ktiles * s.chunks * (long long)p.Bk * p.Hk);
    if (s.fused) {
        p.xtiles = 1;
        hipLaunchKernelGGL((k_ctx_bwd_kv<BF, DP, true>), dim3(kv_blocks), dim3(256), 0, st, p);
    } else {
        p.xtiles = (p.Nq * p.G + 127) / 128;
        hipLaunchKernelGGL((k_ctx_bwd_q<BF, DP>), dim3((unsigned)(p.xtiles * (long long)p.B * p.Hk)), dim3(256), 0, st, p);
        if (!want_kv) return;
        constexpr int shares = DP == 64 ? 1 : 2;
        p.xtiles = s.ktiles * shares;
        if (p.Bk < p.B) hipLaunchKernelGGL((k_ctx_bwd_kv<BF, DP, false, true>), dim3(kv_blocks * shares), dim3(256), 0, st, p);
        else hipLaunchKernelGGL((k_ctx_bwd_kv<BF, DP, false, false>), dim3(kv_blocks * shares), dim3(256), 0, st, p);
    }
    if (s.chunks > 1) {
        const long long plane = (long long)p.Bk * p.Nk * p.Hk * p.d;
        hipLaunchKernelGGL((k_ctx_bwd_sum<BF>), dim3((unsigned)((plane / 4 + 255) / 256), 2), dim3(256), 0, st, p.part, s.chunks, plane, p.dk, p.dv);
    }
}

// (sample, row, head) strides; a tile of 64 rows has to lie within 2^31 bytes
bool row_strides_ok(const void* p, long long a, long long b, long long c) {
    return ((uintptr_t)p % 16) == 0 && a % 8 == 0 && b % 8 == 0 && c % 8 == 0 && b >= 0 && b < (1ll << 24);
}

int check_sizes(const char* name, int dtype, int B, int Nq, int Np, int Nk, int H, int Hk, int d, float scale) {
    VS_REQUIRE(dtype == 1 || dtype == 2, "%s: dtype %d (1 fp16, 2 bf16)", name, dtype);
    VS_REQUIRE(B >= 1 && B <= 65535 && Nq >= 1 && Np >= 0 && Nk >= 0 && Nq <= (1 << 28) && Np <= (1 << 28) && Nk <= (1 << 28), "%s: B=%d Nq=%d Np=%d Nk=%d", name, B, Nq, Np, Nk);
    VS_REQUIRE(Hk >= 1 && H >= Hk && H % Hk == 0 && H <= 1024, "%s: %d heads on %d key heads", name, H, Hk);
    VS_REQUIRE(d >= 8 && d <= 128 && d % 8 == 0, "%s: head width %d (a multiple of 8, at most 128)", name, d);
    VS_REQUIRE(scale > 0.f && scale <= 2.0e38f, "%s: scale must be positive and finite, also times log2 e", name);
    // 2^24 blocks of 256 threads are one launch's limit; splits only multiply small grids.  Row numbers are 32-bit, and a last tile's run up to 127 past the last row
    VS_REQUIRE((long long)Nq * (H / Hk) * B <= (1ll << 31) - 256 && (long long)B * Hk * (((long long)Nq * (H / Hk) + 127) / 128) < (1ll << 24), "%s: B=%d Nq=%d H=%d are too many rows",
               name, B, Nq, H);
    return VS_OK;
}

}  // namespace

extern "C" {

int vidseg_context_attention_scratch_kib(int B, int Nq, int Np, int Nk, int H, int Hk, int d) {
    if (check_sizes("context_attention", 1, B, Nq, Np, Nk, H, Hk, d, 1.f)) return -1;
    // for either plan: a context short enough for k_ctx_short has two key tiles at most, which k_ctx_attn does not deal out, so neither leaves partial results
    const Plan s = make_plan(B, Nq, Np, Nk, H, Hk, d, false);
    return (int)(((long long)s.parts * B * Nq * H * (d + 2) * 4 + 1023) / 1024);
}

int vidseg_context_attention_fwd(const void* q, long long q_b, long long q_n, long long q_h, const void* k_prefix, long long kp_n, long long kp_h,
                                 const void* v_prefix, long long vp_n, long long vp_h, const void* k, long long k_b, long long k_n, long long k_h,
                                 const void* v, long long v_b, long long v_n, long long v_h, const int* lens, const void* mask, long long mask_b,
                                 void* out, void* out_lo, float* lse, int dtype, int B, int Nq, int Np, int Nk, int H, int Hk, int d, float scale, int causal,
                                 void* scratch, long long scratch_kib, hipStream_t st) {
    const int rc = check_sizes("context_attention", dtype, B, Nq, Np, Nk, H, Hk, d, scale);
    if (rc) return rc;
    VS_REQUIRE(q && out && (Nk == 0 || (k && v)) && (Np == 0 || (k_prefix && v_prefix)), "context_attention: null operand");
    VS_REQUIRE(row_strides_ok(q, q_b, q_n, q_h) && row_strides_ok(out, 0, 0, 0) && row_strides_ok(out_lo, 0, 0, 0) && (Nk == 0 || (row_strides_ok(k, k_b, k_n, k_h) && row_strides_ok(v, v_b, v_n, v_h))) &&
                   (Np == 0 || (row_strides_ok(k_prefix, 0, kp_n, kp_h) && row_strides_ok(v_prefix, 0, vp_n, vp_h))),
               "context_attention: operands must be 16-byte aligned with strides that are multiples of 8 elements (rows below 2^24 apart)");
    VS_REQUIRE(!(causal && mask), "context_attention: a causal call takes no key mask");
    const Plan s = make_plan(B, Nq, Np, Nk, H, Hk, d, !causal && !out_lo);
    const long long total = (long long)B * Nq * H;
    const long long need = ((long long)s.parts * total * (d + 2) * 4 + 1023) / 1024;
    VS_REQUIRE(need == 0 || (scratch && scratch_kib >= need), "context_attention: scratch of %lld KiB, needs %lld", scratch_kib, need);
    AttnArgs p{};
    p.q = (const u16*)q; p.q_b = q_b; p.q_n = q_n; p.q_h = q_h;
    p.kp = (const u16*)k_prefix; p.kp_n = kp_n; p.kp_h = kp_h; p.vp = (const u16*)v_prefix; p.vp_n = vp_n; p.vp_h = vp_h;
    p.k = (const u16*)k; p.k_b = k_b; p.k_n = k_n; p.k_h = k_h; p.v = (const u16*)v; p.v_b = v_b; p.v_n = v_n; p.v_h = v_h;
    p.lens = lens; p.mask = (const unsigned char*)mask; p.mask_b = mask_b; p.o = (u16*)out; p.o_lo = (u16*)out_lo; p.lse = lse;
    p.B = B; p.Nq = Nq; p.Np = Np; p.Nk = Nk; p.H = H; p.Hk = Hk; p.G = H / Hk; p.d = d; p.causal = causal; p.c = scale * LOG2E;
    if (s.parts) {
        p.po = (float*)scratch;
        p.pml = p.po + s.parts * total * d;
    }
    if (dtype == 2) {
        if (d <= 64) launch_fwd<true, 64>(p, s, st);
        else if (d <= 96) launch_fwd<true, 96>(p, s, st);
        else launch_fwd<true, 128>(p, s, st);
    } else {
        if (d <= 64) launch_fwd<false, 64>(p, s, st);
        else if (d <= 96) launch_fwd<false, 96>(p, s, st);
        else launch_fwd<false, 128>(p, s, st);
    }
    VS_CHECK_LAUNCH("context_attention");
    return VS_OK;
}

int vidseg_context_attention_bwd_scratch_kib(int B, int Bk, int Nq, int Nk, int H, int Hk, int d) {
    if (check_sizes("context_attention_bwd", 1, B, Nq, 0, Nk, H, Hk, d, 1.f) || (Bk != 1 && Bk != B)) return -1;
    const BwdPlan s = make_bwd_plan(B, Bk, Nq, Nk, H, Hk, d);
    return (int)(((s.delta_floats + s.part_floats) * 4 + 1023) / 1024);
}

int vidseg_context_attention_bwd(const void* dout, long long g_b, long long g_n, long long g_h, const void* q, long long q_b, long long q_n, long long q_h,
                                 const void* k, long long k_b, long long k_n, long long k_h, const void* v, long long v_b, long long v_n,
                                 long long v_h, const int* lens, const void* mask, long long mask_b, const void* out, const void* out_lo, const float* lse, void* dq, void* dk,
                                 void* dv, int dtype, int B, int Bk, int Nq, int Nk, int H, int Hk, int d, float scale, void* scratch,
                                 long long scratch_kib, hipStream_t st) {
    const int rc = check_sizes("context_attention_bwd", dtype, B, Nq, 0, Nk, H, Hk, d, scale);
    if (rc) return rc;
    VS_REQUIRE(Nk >= 1 && (Bk == 1 || Bk == B), "context_attention_bwd: Nk=%d, %d samples of k for %d", Nk, Bk, B);
    VS_REQUIRE(dout && q && k && v && lse && dq && (!dk == !dv), "context_attention_bwd: null operand");
    VS_REQUIRE(row_strides_ok(dout, g_b, g_n, g_h) && row_strides_ok(q, q_b, q_n, q_h) && row_strides_ok(k, k_b, k_n, k_h) && row_strides_ok(v, v_b, v_n, v_h) &&
                   row_strides_ok(out, 0, 0, 0) && row_strides_ok(out_lo, 0, 0, 0) && row_strides_ok(dq, 0, 0, 0) && row_strides_ok(dk, 0, 0, 0) && row_strides_ok(dv, 0, 0, 0),
               "context_attention_bwd: operands must be 16-byte aligned with strides that are multiples of 8 elements (rows below 2^24 apart)");
    const BwdPlan s = make_bwd_plan(B, Bk, Nq, Nk, H, Hk, d);
    VS_REQUIRE((long long)s.ktiles * s.chunks * Bk * Hk < (1ll << 23), "context_attention_bwd: Nk=%d, Hk=%d are too many blocks", Nk, Hk);
    VS_REQUIRE(s.fused || (out && out_lo), "context_attention_bwd: null operand (over 128 keys the forward result and what its rounding left are needed)");
    VS_REQUIRE(dk || !s.fused, "context_attention_bwd: up to 128 keys all three gradients come out of one pass");
    const long long need = ((s.delta_floats + s.part_floats) * 4 + 1023) / 1024;
    VS_REQUIRE(need == 0 || (scratch && scratch_kib >= need), "context_attention_bwd: scratch of %lld KiB, needs %lld", scratch_kib, need);
    BwdArgs p{};
    p.q = (const u16*)q; p.q_b = q_b; p.q_n = q_n; p.q_h = q_h; p.k = (const u16*)k; p.k_b = k_b; p.k_n = k_n; p.k_h = k_h;
    p.v = (const u16*)v; p.v_b = v_b; p.v_n = v_n; p.v_h = v_h; p.go = (const u16*)dout; p.g_b = g_b; p.g_n = g_n; p.g_h = g_h;
    p.o = (const u16*)out; p.o_lo = (const u16*)out_lo; p.lse = lse; p.delta = (float*)scratch; p.lens = lens; p.mask = (const unsigned char*)mask; p.mask_b = mask_b;
    p.dq = (u16*)dq; p.dk = (u16*)dk; p.dv = (u16*)dv; p.part = s.part_floats ? (float*)scratch + s.delta_floats : nullptr;
    p.B = B; p.Bk = Bk; p.Nq = Nq; p.Nk = Nk; p.H = H; p.Hk = Hk; p.G = H / Hk; p.d = d; p.c = scale * LOG2E; p.scale = scale;
    p.chunks = s.chunks; p.per_chunk = s.per_chunk;
    if (dtype == 2) {
        if (d <= 64) launch_bwd<true, 64>(p, s, dk != nullptr, st);
        else if (d <= 96) launch_bwd<true, 96>(p, s, dk != nullptr, st);
        else launch_bwd<true, 128>(p, s, dk != nullptr, st);
    } else {
        if (d <= 64) launch_bwd<false, 64>(p, s, dk != nullptr, st);
        else if (d <= 96) launch_bwd<false, 96>(p, s, dk != nullptr, st);
        else launch_bwd<false, 128>(p, s, dk != nullptr, st);
    }
    VS_CHECK_LAUNCH("context_attention_bwd");
    return VS_OK;
}

}  // extern "C"
