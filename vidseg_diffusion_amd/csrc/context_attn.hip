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

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

template <bool BF> __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {      // 32x32x16
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <bool BF> __device__ __forceinline__ unsigned pack2(float lo, float hi) {           // one rounding to nearest even each
    if constexpr (BF) return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{lo, hi}, b2));
    else return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{lo, hi}, h2));
}
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

struct AttnArgs {
    const u16 *q, *kp, *vp, *k, *v;
    long long q_b, q_n, q_h, kp_n, kp_h, vp_n, vp_h, k_b, k_n, k_h, v_b, v_n, v_h;      // element strides
    const int* lens;
    const unsigned char* mask;
    long long mask_b;
    u16* o;                    // [B][Nq][H][d]
    float* lse;                // [B][H][Nq] or null
    float *po, *pml;           // partial results: [split][B * Nq * H][d], [..][2] = (maximum in log2 units, sum)
    int B, Nq, Np, Nk, H, Hk, G, d, causal;
    float c;                   // scale * log2 e
    int splits, per_split, split0;     // key tiles are dealt out in runs of per_split; the partial results start at index split0
    int xtiles;                // row tiles of a key head
    int stacked;               // rows run over (sample, query, head of the group) and see the prefix only
};

// One row (query, head) per accumulator column.  rows of a key head: r = (sample, query, head of its group), heads fastest.
struct Row {
    int b, qi, h;
    bool on;
};
__device__ __forceinline__ Row row_of(const AttnArgs& p, int b, int hk, long long r, long long rows) {
    Row x;
    x.on = r < rows;
    if (!x.on) r = rows - 1;
    const int per = p.Nq * p.G;
    const int bb = p.stacked ? (int)(r / per) : 0, rem = (int)(r - (long long)bb * per);
    x.b = b + bb;
    x.qi = rem / p.G;
    x.h = hk * p.G + rem % p.G;
    return x;
}

// Blocks reach the 8 XCDs round-robin by their index: every XCD gets one contiguous run of the (key head, split, row tile) space, so the row
// tiles that read the same keys share them through one L2.
__device__ __forceinline__ void block_of(int xtiles, int& y, int& xt) {
    const unsigned tot = gridDim.x, q = tot / 8, r = tot % 8, xcd = blockIdx.x % 8, idx = blockIdx.x / 8;
    const unsigned id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
    y = (int)(id / xtiles);
    xt = (int)(id % xtiles);
}

// WS false: the block's four waves own 32 QB rows each and share key tiles of 64.  WS true (at most 32 rows): every wave holds the same rows
// and takes 32 of each 128 keys; the four partial results are merged at the end.
template <bool BF, int DP, int QB, bool WS> __global__ void __launch_bounds__(256, (DP == 64 || (QB == 1 && !WS)) ? 2 : 1) k_ctx_attn(AttnArgs p) {
    constexpr int KT = WS ? 128 : 64, SL = DP / 8, NST = KT * SL / 256, NBUF = WS ? 1 : 2, NJ = WS ? 1 : 2, ND = DP / 32;
    __shared__ __attribute__((aligned(16))) u16 sK[NBUF][KT * DP], sV[NBUF][KT * DP];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, hi = lane >> 5;
    int y, xt;
    block_of(p.xtiles, y, xt);
    const int split = y % p.splits;
    y /= p.splits;
    const int hk = y % p.Hk, b = y / p.Hk;                            // stacked: b = 0
    const long long rows = (long long)(p.stacked ? p.B : 1) * p.Nq * p.G;
    const long long r0 = (long long)xt * (WS ? 32 : 128 * QB);
    Row row[QB];
    u32x4 fq[QB][DP / 16];
#pragma unroll
    for (int i = 0; i < QB; ++i) {
        row[i] = row_of(p, b, hk, r0 + (WS ? 0 : wave * 32 * QB) + i * 32 + l31, rows);
        const u16* qp = p.q + row[i].b * p.q_b + row[i].qi * p.q_n + row[i].h * p.q_h;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            const int at = s * 16 + hi * 8;
            fq[i][s] = *reinterpret_cast<const u32x4*>(qp + (at < p.d ? at : 0));
            if (at >= p.d) fq[i][s] = u32x4{0u, 0u, 0u, 0u};
        }
    }
    // the key tiles this block visits: prefix tiles first, then the sample's own
    const int len = p.stacked ? 0 : (p.lens ? max(0, min(p.lens[b], p.Nk)) : p.Nk);
    const long long last_r = (r0 + (WS ? 32 : 128 * QB) < rows ? r0 + (WS ? 32 : 128 * QB) : rows) - 1;
    const int seen = p.causal ? max(0, min(len, len - p.Nq + 1 + (int)(last_r / p.G))) : len;      // own keys that the block's last row sees
    const int all_see = p.causal ? len - p.Nq + 1 + (int)(r0 / p.G) : len;                          // own keys that every row sees
    const int np = p.Np;
    const int T0 = (np + KT - 1) / KT, T1 = (seen + KT - 1) / KT;
    const int tb = min(split * p.per_split, T0 + T1), te = p.splits == 1 ? T0 + T1 : min(tb + p.per_split, T0 + T1);

    u32x4 rk[NST], rv[NST];
    unsigned long long live = 0;                                      // keys of the staged tile that exist (WS: of this wave's 32)
    const u16* kown = p.k + b * p.k_b + hk * p.k_h;
    const u16* vown = p.v + b * p.v_b + hk * p.v_h;
    const unsigned char* mrow = p.mask ? p.mask + b * p.mask_b : nullptr;
    auto load_tile = [&](int t) {
        const bool own = t >= T0;
        const int k0 = (own ? t - T0 : t) * KT, n = own ? seen : np;
        const u16* kb = own ? kown : p.kp + hk * p.kp_h;
        const u16* vb = own ? vown : p.vp + hk * p.vp_h;
        const long long kn = own ? p.k_n : p.kp_n, vn = own ? p.v_n : p.vp_n;
        const unsigned char* mk = own ? mrow : nullptr;
#pragma unroll
        for (int i = 0; i < NST; ++i) {
            const int id = tid + 256 * i, r = id / SL, slot = id % SL, key = k0 + r, kk = min(key, n - 1);
            const bool ok = key < n && slot * 8 < p.d && (!mk || mk[kk]);
            const int at = slot * 8 < p.d ? slot * 8 : 0;
            rk[i] = *reinterpret_cast<const u32x4*>(kb + kk * kn + at);
            rv[i] = *reinterpret_cast<const u32x4*>(vb + kk * vn + at);
            if (!ok) rk[i] = rv[i] = u32x4{0u, 0u, 0u, 0u};
        }
        const int key = k0 + (WS ? wave * 32 + l31 : lane);
        live = __ballot(key < n && (!mk || mk[min(key, n - 1)]));
    };
    auto store_tile = [&](int buf) {
#pragma unroll
        for (int i = 0; i < NST; ++i) {
            const int id = tid + 256 * i, r = id / SL, slot = id % SL;
            *reinterpret_cast<u32x4*>(&sK[buf][slot_at<DP>(r, slot)]) = rk[i];
            *reinterpret_cast<u32x4*>(&sV[buf][slot_at<DP>(r, slot)]) = rv[i];
        }
    };

    f32x16 oacc[QB][ND];
    float m_run[QB], l_run[QB];
#pragma unroll
    for (int i = 0; i < QB; ++i) {
        m_run[i] = -INFINITY;
        l_run[i] = 0.f;
#pragma unroll
        for (int n = 0; n < ND; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) oacc[i][n][r] = 0.f;
    }

    if (tb < te) {
        load_tile(tb);
        store_tile(0);
    }
    __syncthreads();
    for (int t = tb; t < te; ++t) {
        const int buf = NBUF == 2 ? (t - tb) & 1 : 0;
        const unsigned long long now = live;
        if (t + 1 < te) load_tile(t + 1);
        const int k0 = (t >= T0 ? t - T0 : t) * KT + (WS ? wave * 32 : 0);
        const bool edge = p.causal && t >= T0 && k0 + 32 * NJ > all_see;
#pragma unroll
        for (int i = 0; i < QB; ++i) {
            f32x16 s[NJ];
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[j][r] = 0.f;
#pragma unroll
                for (int e = 0; e < DP / 16; ++e)
                    s[j] = mfma<BF>(read_row<DP>(sK[buf], (WS ? wave * 32 : j * 32) + l31, e * 2 + hi), fq[i][e], s[j]);
            }
            if (now != ~0ull || edge) {
                const int lim = edge ? len - p.Nq + row[i].qi - k0 - 4 * hi : 1 << 30;              // keys up to this one (in this lane's numbering) are seen
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const unsigned bits = (unsigned)(now >> (32 * j)) >> (4 * hi);
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int at = (r & 3) + 8 * (r >> 2);
                        if (!((bits >> at) & 1u) || 32 * j + at > lim) s[j][r] = -INFINITY;
                    }
                }
            }
            float mx = s[0][0];
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[j][r]);
            mx = half_max(mx) * p.c;
            const float m_new = fmaxf(m_run[i], mx);
            const float ref = m_new == -INFINITY ? 0.f : m_new;       // a row without a key so far: every exp2 below gives 0
            if (__any(m_new > m_run[i])) {
                const float alpha = __builtin_amdgcn_exp2f(m_run[i] - ref);
                l_run[i] *= alpha;
#pragma unroll
                for (int n = 0; n < ND; ++n)
#pragma unroll
                    for (int r = 0; r < 16; ++r) oacc[i][n][r] *= alpha;
                m_run[i] = m_new;
            }
            float sum = 0.f;
            u32x4 fp[NJ][2];
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(fmaf(s[j][r], p.c, -ref)), p1 = __builtin_amdgcn_exp2f(fmaf(s[j][r + 1], p.c, -ref));
                    sum += p0 + p1;
                    fp[j][r >> 3][(r >> 1) & 3] = pack2<BF>(p0, p1);          // p in (0, 1]: the one rounding of the probabilities
                }
            l_run[i] += half_sum(sum);
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int n = 0; n < ND; ++n)
                        oacc[i][n] = mfma<BF>(read_tr<DP>(sV[buf], (WS ? wave * 32 : j * 32) + e * 16, n * 32, lane), fp[j][e], oacc[i][n]);
        }
        if (NBUF == 1) __syncthreads();
        if (t + 1 < te) store_tile(NBUF == 2 ? buf ^ 1 : 0);
        __syncthreads();
    }

    const long long total = (long long)p.B * p.Nq * p.H;
    if constexpr (WS) {
        // the four waves' results of the same rows: maxima and sums first, then the accumulators through the tile memory (fp32 [wave][row][DP])
        __shared__ float sm[4][32], sl[4][32];
        static_assert(4 * 32 * DP * 4 <= (int)sizeof(sK) + (int)sizeof(sV), "merge buffer");
        float* so = reinterpret_cast<float*>(&sK[0][0]);
        float* so2 = reinterpret_cast<float*>(&sV[0][0]);             // waves 0, 1 use sK, waves 2, 3 use sV
        float* mine = (wave < 2 ? so : so2) + (wave & 1) * 32 * DP;
        if (hi == 0) {
            sm[wave][l31] = m_run[0];
            sl[wave][l31] = l_run[0];
        }
#pragma unroll
        for (int n = 0; n < ND; ++n)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *reinterpret_cast<f32x4*>(mine + l31 * DP + n * 32 + 2 * r + 4 * hi) = f32x4{oacc[0][n][r], oacc[0][n][r + 1], oacc[0][n][r + 2], oacc[0][n][r + 3]};
        __syncthreads();
        const int rr = tid >> 3;
        const Row x = row_of(p, b, hk, r0 + rr, rows);
        if (x.on) {
            float m = -INFINITY, l = 0.f, w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) m = fmaxf(m, sm[i][rr]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[i][rr] - m);
                l += w[i] * sl[i][rr];
            }
            const long long id = ((long long)x.b * p.Nq + x.qi) * p.H + x.h;
            const float inv = l > 0.f ? 1.0f / l : 0.f;
            for (int c = (tid & 7) * 4; c < p.d; c += 32) {
                f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 t = *reinterpret_cast<const f32x4*>((i < 2 ? so : so2) + (i & 1) * 32 * DP + rr * DP + c);
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[e] += w[i] * t[e];
                }
                if (p.po) *reinterpret_cast<f32x4*>(p.po + ((p.split0 + split) * total + id) * p.d + c) = a;
                else *reinterpret_cast<u32x2*>(p.o + id * p.d + c) = u32x2{pack2<BF>(a[0] * inv, a[1] * inv), pack2<BF>(a[2] * inv, a[3] * inv)};
            }
            if ((tid & 7) == 0) {
                if (p.po) *reinterpret_cast<f32x2*>(p.pml + ((p.split0 + split) * total + id) * 2) = f32x2{m, l};
                else if (p.lse) p.lse[((long long)x.b * p.H + x.h) * p.Nq + x.qi] = (m + __builtin_amdgcn_logf(l)) * LN2;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < QB; ++i) {
            if (!row[i].on) continue;
            const long long id = ((long long)row[i].b * p.Nq + row[i].qi) * p.H + row[i].h;
            const float inv = l_run[i] > 0.f ? 1.0f / l_run[i] : 0.f;
#pragma unroll
            for (int n = 0; n < ND; ++n)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const int c = n * 32 + 2 * r + 4 * hi;
                    if (c >= p.d) continue;
                    if (p.po)
                        *reinterpret_cast<f32x4*>(p.po + ((p.split0 + split) * total + id) * p.d + c) = f32x4{oacc[i][n][r], oacc[i][n][r + 1], oacc[i][n][r + 2], oacc[i][n][r + 3]};
                    else
                        *reinterpret_cast<u32x2*>(p.o + id * p.d + c) = u32x2{pack2<BF>(oacc[i][n][r] * inv, oacc[i][n][r + 1] * inv), pack2<BF>(oacc[i][n][r + 2] * inv, oacc[i][n][r + 3] * inv)};
                }
            if (hi == 0) {
                if (p.po) *reinterpret_cast<f32x2*>(p.pml + ((p.split0 + split) * total + id) * 2) = f32x2{m_run[i], l_run[i]};
                else if (p.lse) p.lse[((long long)row[i].b * p.H + row[i].h) * p.Nq + row[i].qi] = (m_run[i] + __builtin_amdgcn_logf(l_run[i])) * LN2;
            }
        }
    }
}

// Joins the partial results of one row: sixteen lanes per row, eight channels each
template <bool BF> __global__ void __launch_bounds__(256) k_ctx_join(const float* __restrict__ po, const float* __restrict__ pml, int splits, long long total, int d,
                                                                   int Nq, int H, u16* __restrict__ o, float* __restrict__ lse) {
    const long long id = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int c = (threadIdx.x & 15) * 8;
    if (id >= total) return;
    float m = -INFINITY, l = 0.f;
    for (int s = 0; s < splits; ++s) m = fmaxf(m, pml[(s * total + id) * 2]);
    float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (m != -INFINITY)
        for (int s = 0; s < splits; ++s) {
            const f32x2 x = *reinterpret_cast<const f32x2*>(pml + (s * total + id) * 2);
            if (x[0] == -INFINITY) continue;
            const float w = __builtin_amdgcn_exp2f(x[0] - m);
            l += w * x[1];
            if (c < d) {
                const f32x4 t0 = *reinterpret_cast<const f32x4*>(po + (s * total + id) * d + c), t1 = *reinterpret_cast<const f32x4*>(po + (s * total + id) * d + c + 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    a[e] += w * t0[e];
                    a[e + 4] += w * t1[e];
                }
            }
        }
    const float inv = l > 0.f ? 1.0f / l : 0.f;
    if (c < d)
        *reinterpret_cast<u32x4*>(o + id * d + c) = u32x4{pack2<BF>(a[0] * inv, a[1] * inv), pack2<BF>(a[2] * inv, a[3] * inv), pack2<BF>(a[4] * inv, a[5] * inv), pack2<BF>(a[6] * inv, a[7] * inv)};
    if (lse && c == 0) {
        const long long bq = id / H;
        lse[((bq / Nq) * H + id % H) * Nq + bq % Nq] = (m + __builtin_amdgcn_logf(l)) * LN2;
    }
}

// How a call is laid out: which rows a block owns, how the keys are dealt out, which launches that takes
struct Plan {
    bool few;                  // own keys: at most 32 rows per key head, waves split the keys
    bool stack;                // prefix: rows of all samples stacked (a row tile of one sample alone would be mostly empty)
    bool stack_few;
    int own_splits, own_per, pre_splits, pre_per;
    int parts;                 // partial results to join (0: the kernel writes the result)
};
Plan make_plan(int B, int Nq, int Np, int Nk, int H, int Hk) {
    Plan s{};
    const int G = H / Hk;
    const long long rows = (long long)Nq * G;
    s.few = rows <= 32;
    s.stack = Np > 0 && rows < 128;
    s.stack_few = s.stack && rows * B <= 32;
    const int kt = s.few ? 128 : 64;
    const long long blocks = (long long)B * Hk * (s.few ? 1 : (rows + 127) / 128);
    const int tiles = (Nk + kt - 1) / kt + (s.stack ? 0 : (Np + kt - 1) / kt);
    auto deal = [](long long blocks, int tiles, int least, int& splits, int& per) {      // about 512 blocks, at least `least` tiles each
        const long long want = blocks >= 384 ? 1 : (512 + blocks - 1) / blocks;
        per = (int)((tiles + want - 1) / want);
        if (per < least) per = least;
        splits = tiles > per ? (tiles + per - 1) / per : 1;
        if (splits == 1) per = tiles > 0 ? tiles : 1;
    };
    deal(blocks, tiles, s.few ? 2 : 4, s.own_splits, s.own_per);
    if (s.stack) {
        const int pk = s.stack_few ? 128 : 64;
        deal((long long)Hk * ((rows * B + 127) / 128), (Np + pk - 1) / pk, s.stack_few ? 2 : 4, s.pre_splits, s.pre_per);
    }
    const int own = Nk > 0 || !s.stack ? s.own_splits : 0;
    s.parts = own + (s.stack ? s.pre_splits : 0);
    if (s.parts <= 1) s.parts = 0;
    return s;
}

template <bool BF, int DP> void launch_one(const AttnArgs& p, bool ws, dim3 grid, hipStream_t st) {
    if (ws) hipLaunchKernelGGL((k_ctx_attn<BF, DP, 1, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((k_ctx_attn<BF, DP, 1, false>), grid, dim3(256), 0, st, p);
}
void launch_attn(AttnArgs p, int dtype, bool ws, long long tiles, long long heads, hipStream_t st) {
    p.xtiles = (int)tiles;
    const dim3 grid((unsigned)(tiles * heads * p.splits));
    if (dtype == 2) {
        if (p.d <= 64) launch_one<true, 64>(p, ws, grid, st);
        else if (p.d <= 96) launch_one<true, 96>(p, ws, grid, st);
        else launch_one<true, 128>(p, ws, grid, st);
    } else {
        if (p.d <= 64) launch_one<false, 64>(p, ws, grid, st);
        else if (p.d <= 96) launch_one<false, 96>(p, ws, grid, st);
        else launch_one<false, 128>(p, ws, grid, st);
    }
}

bool row_strides_ok(const void* p, long long a, long long b, long long c) { return ((uintptr_t)p % 16) == 0 && a % 8 == 0 && b % 8 == 0 && c % 8 == 0; }

int check_sizes(const char* name, int dtype, int B, int Nq, int Np, int Nk, int H, int Hk, int d, float scale) {
    VS_REQUIRE(dtype == 1 || dtype == 2, "%s: dtype %d (1 fp16, 2 bf16)", name, dtype);
    VS_REQUIRE(B >= 1 && B <= 65535 && Nq >= 1 && Np >= 0 && Nk >= 0 && Nq <= (1 << 28) && Np <= (1 << 28) && Nk <= (1 << 28), "%s: B=%d Nq=%d Np=%d Nk=%d", name, B, Nq, Np, Nk);
    VS_REQUIRE(Hk >= 1 && H >= Hk && H % Hk == 0 && H <= 1024, "%s: %d heads on %d key heads", name, H, Hk);
    VS_REQUIRE(d >= 8 && d <= 128 && d % 8 == 0, "%s: head width %d (a multiple of 8, at most 128)", name, d);
    VS_REQUIRE(scale > 0.f && scale <= 3.0e38f, "%s: scale must be positive and finite", name);
    // 2^24 blocks of 256 threads are one launch's limit; splits only multiply small grids
    VS_REQUIRE((long long)Nq * (H / Hk) * B < (1ll << 31) && (long long)B * Hk * (((long long)Nq * (H / Hk) + 127) / 128) < (1ll << 24), "%s: B=%d Nq=%d H=%d are too many rows",
               name, B, Nq, H);
    return VS_OK;
}

}  // namespace

extern "C" {

int vidseg_context_attention_scratch_kib(int B, int Nq, int Np, int Nk, int H, int Hk, int d) {
    if (check_sizes("context_attention", 1, B, Nq, Np, Nk, H, Hk, d, 1.f)) return -1;
    const Plan s = make_plan(B, Nq, Np, Nk, H, Hk);
    return (int)(((long long)s.parts * B * Nq * H * (d + 2) * 4 + 1023) / 1024);
}

int vidseg_context_attention_fwd(const void* q, long long q_b, long long q_n, long long q_h, const void* k_prefix, long long kp_n, long long kp_h,
                                 const void* v_prefix, long long vp_n, long long vp_h, const void* k, long long k_b, long long k_n, long long k_h,
                                 const void* v, long long v_b, long long v_n, long long v_h, const int* lens, const void* mask, long long mask_b,
                                 void* out, float* lse, int dtype, int B, int Nq, int Np, int Nk, int H, int Hk, int d, float scale, int causal,
                                 void* scratch, long long scratch_kib, hipStream_t st) {
    const int rc = check_sizes("context_attention", dtype, B, Nq, Np, Nk, H, Hk, d, scale);
    if (rc) return rc;
    VS_REQUIRE(q && out && (Nk == 0 || (k && v)) && (Np == 0 || (k_prefix && v_prefix)), "context_attention: null operand");
    VS_REQUIRE(row_strides_ok(q, q_b, q_n, q_h) && row_strides_ok(out, 0, 0, 0) && (Nk == 0 || (row_strides_ok(k, k_b, k_n, k_h) && row_strides_ok(v, v_b, v_n, v_h))) &&
                   (Np == 0 || (row_strides_ok(k_prefix, 0, kp_n, kp_h) && row_strides_ok(v_prefix, 0, vp_n, vp_h))),
               "context_attention: operands must be 16-byte aligned with strides that are multiples of 8 elements");
    VS_REQUIRE(!(causal && mask), "context_attention: a causal call takes no key mask");
    const Plan s = make_plan(B, Nq, Np, Nk, H, Hk);
    const long long total = (long long)B * Nq * H;
    const long long need = ((long long)s.parts * total * (d + 2) * 4 + 1023) / 1024;
    VS_REQUIRE(need == 0 || (scratch && scratch_kib >= need), "context_attention: scratch of %lld KiB, needs %lld", scratch_kib, need);
    AttnArgs p{};
    p.q = (const u16*)q; p.q_b = q_b; p.q_n = q_n; p.q_h = q_h;
    p.kp = (const u16*)k_prefix; p.kp_n = kp_n; p.kp_h = kp_h; p.vp = (const u16*)v_prefix; p.vp_n = vp_n; p.vp_h = vp_h;
    p.k = (const u16*)k; p.k_b = k_b; p.k_n = k_n; p.k_h = k_h; p.v = (const u16*)v; p.v_b = v_b; p.v_n = v_n; p.v_h = v_h;
    p.lens = lens; p.mask = (const unsigned char*)mask; p.mask_b = mask_b; p.o = (u16*)out; p.lse = lse;
    p.B = B; p.Nq = Nq; p.Np = Np; p.Nk = Nk; p.H = H; p.Hk = Hk; p.G = H / Hk; p.d = d; p.causal = causal; p.c = scale * LOG2E;
    if (s.parts) {
        p.po = (float*)scratch;
        p.pml = p.po + s.parts * total * d;
    }
    const long long rows = (long long)Nq * p.G;
    if (s.stack) {
        AttnArgs a = p;
        a.stacked = 1; a.splits = s.pre_splits; a.per_split = s.pre_per; a.split0 = 0; a.Nk = 0; a.causal = 0; a.lens = nullptr; a.mask = nullptr;
        launch_attn(a, dtype, s.stack_few, s.stack_few ? 1 : (rows * B + 127) / 128, Hk, st);
        p.Np = 0;
        p.split0 = s.pre_splits;
    }
    if (Nk > 0 || !s.stack) {
        p.splits = s.own_splits; p.per_split = s.own_per;
        launch_attn(p, dtype, s.few, s.few ? 1 : (rows + 127) / 128, (long long)B * Hk, st);
    }
    if (s.parts) {
        const unsigned blocks = (unsigned)((total + 15) / 16);
        if (dtype == 2) hipLaunchKernelGGL((k_ctx_join<true>), dim3(blocks), dim3(256), 0, st, p.po, p.pml, s.parts, total, d, Nq, H, p.o, lse);
        else hipLaunchKernelGGL((k_ctx_join<false>), dim3(blocks), dim3(256), 0, st, p.po, p.pml, s.parts, total, d, Nq, H, p.o, lse);
    }
    VS_CHECK_LAUNCH("context_attention");
    return VS_OK;
}

}  // extern "C"
