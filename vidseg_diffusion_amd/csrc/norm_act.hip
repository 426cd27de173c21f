// HIPCC_FLAGS: -fno-slp-vectorize -Xclang -target-feature -Xclang -packed-fp32-ops
// GroupNorm with an optional SiLU on channels-last maps x [B][HW][C], forward and backward, fp32 / fp16 / bf16 storage.
//
//   xh = (x - mean_g) * rstd_g,  z = xh * gamma + beta,  y = z or z * sigmoid(z)
//   dz = dy * act'(z),  dbeta = sum dz,  dgamma = sum dz * xh,
//   dx = rstd_g * (gamma * dz - (mean over the group of gamma * dz) - xh * (mean over the group of gamma * dz * xh))
//
// Everything is held in fp32 between the load and the one rounding of the store.  A thread owns VEC neighbouring channels (16 bytes) of
// every R-th row, so a wave reads whole rows; sums go channel -> group only after the rows are summed, so any C / G works, also
// groups that end inside a 16-byte piece (320 channels in 32 groups of 10).  Two launches forward (chunk statistics; merge and apply) and
// two backward (channel and group sums of a chunk; merge and dx, with dgamma and dbeta in extra blocks): no atomics, every sum has one order.
// A chunk's row count depends on HW and C only, so a sample's result does not depend on the batch it is in.
//
// What bounds it: bytes.  28 x 64 x 64 x 320 fp16: statistics 17.8 us (73 MB read, 4.1 TB/s), apply 28.4 us (147 MB, 5.2 TB/s; a large copy reaches 5.1);
// 14 x 32 x 32 x 1920 bf16 with SiLU, backward: sums 28.7 us (110 MB; exp2 and rcp of every value are most of it: without SiLU 22), dx 31.3 us (165 MB,
// 5.3 TB/s).  x (and dy) are read twice, the second time out of the last-level cache: a block owns a run of rows, so a group's statistics need every block of
// its sample.  (A block that owned whole groups -- 80 KB each at 64 x 64 x 320 -- could keep them on its CU and read x once; that form is not here.)
// Deeper unrolling of either pass changed nothing; 28 x 4096 x 320 and 14 x 1024 x 1920 take 51 / 40 us at 40 K values a chunk, 49 / 47 at 20 K, 63 / 53 at 80 K.
#include "common.h"

namespace {

constexpr int NT = 256;
typedef float f32x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Stored;
template <> struct Stored<float> {
    typedef float type;
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
};
template <> struct Stored<_Float16> {
    typedef _Float16 type;
    static __device__ __forceinline__ float up(_Float16 v) { return (float)v; }
    static __device__ __forceinline__ _Float16 down(float v) { return (_Float16)v; }
};
template <> struct Stored<__bf16> {
    typedef __bf16 type;
    static __device__ __forceinline__ float up(__bf16 v) { return (float)v; }
    static __device__ __forceinline__ __bf16 down(float v) { return (__bf16)v; }
};

template <typename T, int VEC> __device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) {
    typedef T vec __attribute__((ext_vector_type(VEC)));
    if constexpr (VEC == 1) {
        v[0] = Stored<T>::up(*p);
    } else {
        const vec r = *reinterpret_cast<const vec*>(p);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = Stored<T>::up(r[e]);
    }
}
template <typename T, int VEC> __device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
    typedef T vec __attribute__((ext_vector_type(VEC)));
    if constexpr (VEC == 1) {
        *p = Stored<T>::down(v[0]);
    } else {
        vec r;
#pragma unroll
        for (int e = 0; e < VEC; ++e) r[e] = Stored<T>::down(v[e]);
        *reinterpret_cast<vec*>(p) = r;
    }
}

__device__ __forceinline__ float sigmoid_f32(float z) {           // exp2 overflows to inf for z < -128 / log2 e: 1 / inf = 0, the limit
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896340736f));
}

struct NormArgs {
    const void* x;
    long long x_b, x_row;                 // element strides of a sample and of a row
    const void* dy;
    long long dy_b, dy_row;
    long long HW;
    int B, C, G, rows, nchunk, act;
    float eps, down;                      // down: exact factor of every M2
    const float *gamma, *beta;
    void* out;                            // y or dx, contiguous [B][HW][C]
    float *mean, *rstd;                   // [B][G]
    float* part;                          // [B][nchunk][G][2]; forward (mean, M2 * down) of a group over a chunk, backward its sums of gamma * dz and gamma * dz * xh
    float* chan;                          // backward: [B][nchunk][2][C] sums of dz and dz * xh over a chunk
    float *dgamma, *dbeta;
};

// Sums over the R row lanes of a column pass: s[k][j] over j = 0..R-1 laid out [R][cols * VEC] in LDS; afterwards row 0 holds the totals.
// (all NT threads call it)
template <int VEC> __device__ __forceinline__ void fold_rows(float* s0, float* s1, int R, int width) {
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += NT) {
        float a = s0[c], b = s1[c];
        for (int j = 1; j < R; ++j) {
            a += s0[j * width + c];
            b += s1[j * width + c];
        }
        s0[c] = a;
        s1[c] = b;
    }
    __syncthreads();
}

// Lanes that share the work of one group: a power of two up to a wave's 64, so that G * lanes fills the block
__device__ __forceinline__ int lanes_per(int G) {
    int l = 1;
    while (l < 64 && G * l * 2 <= NT) l *= 2;
    return l;
}
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// ---- forward, launch 1: (mean, M2) of every group over the rows of one chunk, M2 the sum of squared deviations from that mean.
// A thread takes its rows less the first of them, x - k, and carries mean and M2 along: with d = (x - k) - mean,  mean += d / n,  M2 += d ((x - k) - mean);
// row lanes, channels and chunks are then merged by theirs:
//   mean = mean_a + (mean_b - mean_a) n_b / n,   M2 = M2_a + M2_b + (mean_b - mean_a)^2 n_a n_b / n.
// No difference of large squares anywhere, so a map whose mean is far from zero, or whose first rows lie far from the others, keeps its variance.  M2 is n times the
// variance, and fp32 would not hold it for maps whose variance it holds: it is carried times 2^-32 (exact; every bit is as without), except where eps is below 2^-60
// and a small M2's bits that this costs (variances of 2^-94 and less) would count.  Channel means are summed times 2^-13, the most there are, for the same reason.
// (Sums of x - k and its square would take 3 operations a value for 5, and lose a factor of the rows where the first one is an outlier.)
template <typename T, int VEC> __global__ void __launch_bounds__(NT) k_gna_stats(NormArgs p) {
    extern __shared__ float lds[];
    const int C = p.C, cols = C / VEC, b = blockIdx.y, chunk = blockIdx.x;
    const int pc = cols < NT ? cols : NT, R = NT / pc, width = pc * VEC;
    float* ch_mean = lds;                 // [C]
    float* ch_m2 = lds + C;               // [C]
    float* s0 = lds + 2 * C;              // [R][width] means of the row lanes
    float* s1 = s0 + R * width;           // ... and M2
    constexpr float MEANS = 1.220703125e-4f;
    const long long r0 = (long long)chunk * p.rows;
    const int n = (int)(p.HW - r0 < p.rows ? p.HW - r0 : p.rows);
    const T* x = (const T*)p.x + b * p.x_b + r0 * p.x_row;
    const int col = threadIdx.x % pc, rl = threadIdx.x / pc;
    for (int c0 = 0; c0 < cols; c0 += pc) {
        if (rl < R && rl < n && c0 + col < cols) {
            float k[VEC], a[VEC], q[VEC], count = 1.f;
            const T* xc = x + (long long)(c0 + col) * VEC;
            load_vec<T, VEC>(xc + rl * p.x_row, k);
#pragma unroll
            for (int e = 0; e < VEC; ++e) a[e] = q[e] = 0.f;
#pragma unroll 4
            for (int r = rl + R; r < n; r += R) {
                float v[VEC];
                load_vec<T, VEC>(xc + r * p.x_row, v);
                count += 1.f;
                const float inv = __builtin_amdgcn_rcpf(count);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float u = v[e] - k[e], d = u - a[e];
                    a[e] += d * inv;
                    q[e] += d * (u - a[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                s0[rl * width + col * VEC + e] = k[e] + a[e];
                s1[rl * width + col * VEC + e] = q[e] * p.down;
            }
        }
        __syncthreads();
        const int w = (cols - c0 < pc ? cols - c0 : pc) * VEC, lanes = R < n ? R : n;
        for (int c = threadIdx.x; c < w; c += NT) {                 // lane j has (n - j) / R rows, rounded up
            const float k = s0[c];
            float s = 0.f, m2 = 0.f;
            for (int j = 1; j < lanes; ++j) s += (float)((n - j + R - 1) / R) * (s0[j * width + c] - k);
            const float m = s / (float)n;                           // about lane 0's mean
            for (int j = 0; j < lanes; ++j) {
                const float d = s0[j * width + c] - k - m;
                m2 += s1[j * width + c] + (float)((n - j + R - 1) / R) * p.down * d * d;
            }
            ch_mean[c0 * VEC + c] = k + m;
            ch_m2[c0 * VEC + c] = m2;
        }
        __syncthreads();
    }
    const int cg = C / p.G, lanes = lanes_per(p.G), sub = threadIdx.x % lanes, stride = NT / lanes;
    for (int g0 = 0; g0 < p.G; g0 += stride) {                      // whole waves take part in the shuffles; lanes past G work on the last group
        const int g = min(g0 + (int)threadIdx.x / lanes, p.G - 1);
        float m = 0.f, m2 = 0.f;
        for (int c = sub; c < cg; c += lanes) m += ch_mean[g * cg + c] * MEANS;
        m = lanes_sum(m, lanes) / ((float)cg * MEANS);
        for (int c = sub; c < cg; c += lanes) {
            const float d = ch_mean[g * cg + c] - m;
            m2 += ch_m2[g * cg + c] + (float)n * p.down * d * d;
        }
        m2 = lanes_sum(m2, lanes);
        if (sub == 0) *reinterpret_cast<f32x2*>(p.part + (((long long)b * p.nchunk + chunk) * p.G + g) * 2) = f32x2{m, m2};
    }
}

// rows n_b of mean m_b and M2 m2_b (over cg channels, times down) into (n, m, m2); either may be empty (a mean of 0, from which the other's may lie further than a
// square can hold)
__device__ __forceinline__ void merge(float& n, float& m, float& m2, float n_b, float m_b, float m2_b, float cg, float down) {
    const float all = n + n_b, share = n > 0.f ? n_b * __builtin_amdgcn_rcpf(all) : 1.f, d = m_b - m;      // (the first part is taken as it is)
    const float both = n * share, d0 = both > 0.f ? d : 0.f;
    m += d * share;
    m2 += m2_b + d0 * down * d0 * both * cg;
    n = all;
}

// ---- forward, launch 2: every block merges its sample's chunk statistics and writes one chunk of y.  Those are 8 bytes a group and chunk out of L2, 8 KB at 64 x 64 x 320
// (32 chunks); chunks do not grow with the map, so what all blocks read of them grows with its square: 210 KB a block at 512 x 512 x 128 (820 chunks), beside 82 KB of x
template <typename T, int VEC> __global__ void __launch_bounds__(NT) k_gna_apply(NormArgs p) {
    extern __shared__ float lds[];
    const int C = p.C, cols = C / VEC, b = blockIdx.y, chunk = blockIdx.x, cg = C / p.G;
    float* g_mean = lds;
    float* g_rstd = lds + p.G;
    const int lanes = lanes_per(p.G), sub = threadIdx.x % lanes, stride = NT / lanes;
    for (int g0 = 0; g0 < p.G; g0 += stride) {
        const int g = min(g0 + (int)threadIdx.x / lanes, p.G - 1);
        const f32x2* o = reinterpret_cast<const f32x2*>(p.part) + (long long)b * p.nchunk * p.G + g;
        float n = 0.f, m = 0.f, m2 = 0.f;                           // rows (exact below 2^24 a lane), mean and M2 of this lane's chunks
#pragma unroll 4
        for (int i = sub; i < p.nchunk; i += lanes) {
            const float rows = (float)(i + 1 < p.nchunk ? p.rows : (int)(p.HW - (long long)i * p.rows));
            const f32x2 t = o[(long long)i * p.G];
            merge(n, m, m2, rows, t[0], t[1], (float)cg, p.down);
        }
        for (int w = 1; w < lanes; w *= 2) {
            const float n_b = __shfl_xor(n, w, 64), m_b = __shfl_xor(m, w, 64), m2_b = __shfl_xor(m2, w, 64);
            // the lower lane's part first: both lanes get the same values
            const bool up = sub & w;
            float n_a = up ? n_b : n, m_a = up ? m_b : m, m2_a = up ? m2_b : m2;
            merge(n_a, m_a, m2_a, up ? n : n_b, up ? m : m_b, up ? m2 : m2_b, (float)cg, p.down);
            n = n_a;
            m = m_a;
            m2 = m2_a;
        }
        const float rstd = 1.0f / sqrtf(m2 / ((float)p.HW * (float)cg * p.down) + p.eps);
        if (sub == 0) {
            g_mean[g] = m;
            g_rstd[g] = rstd;
            if (p.mean && chunk == 0) {
                p.mean[(long long)b * p.G + g] = m;
                p.rstd[(long long)b * p.G + g] = rstd;
            }
        }
    }
    __syncthreads();
    const int pc = cols < NT ? cols : NT, R = NT / pc;
    const long long r0 = (long long)chunk * p.rows;
    const int n = (int)(p.HW - r0 < p.rows ? p.HW - r0 : p.rows);
    const int col = threadIdx.x % pc, rl = threadIdx.x / pc;
    if (rl >= R) return;
    for (int c = col; c < cols; c += pc) {
        float mean[VEC], scale[VEC], shift[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int ch = c * VEC + e, g = ch / cg;
            mean[e] = g_mean[g];
            scale[e] = g_rstd[g] * p.gamma[ch];
            shift[e] = p.beta[ch];
        }
        const T* x = (const T*)p.x + b * p.x_b + r0 * p.x_row + (long long)c * VEC;
        T* y = (T*)p.out + ((long long)b * p.HW + r0) * C + (long long)c * VEC;
#pragma unroll 4
        for (int r = rl; r < n; r += R) {
            float v[VEC];
            load_vec<T, VEC>(x + r * p.x_row, v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float z = (v[e] - mean[e]) * scale[e] + shift[e];
                v[e] = p.act ? z * sigmoid_f32(z) : z;
            }
            store_vec<T, VEC>(y + (long long)r * C, v);
        }
    }
}

// dz of one value: act' (z) = sig (1 + z (1 - sig))
__device__ __forceinline__ float dz_of(float dy, float z, int act) {
    if (!act) return dy;
    const float s = sigmoid_f32(z);
    return dy * (s * (1.0f + z * (1.0f - s)));
}

// ---- backward, launch 1: over the rows of one chunk, per channel the sums of dz and dz * xh, and from them per group those of gamma * dz, gamma * dz * xh
template <typename T, int VEC> __global__ void __launch_bounds__(NT) k_gna_bwd_sums(NormArgs p) {
    extern __shared__ float lds[];
    const int C = p.C, cols = C / VEC, b = blockIdx.y, chunk = blockIdx.x, cg = C / p.G;
    const int pc = cols < NT ? cols : NT, R = NT / pc, width = pc * VEC;
    float* ch0 = lds;                     // [C] gamma * sums
    float* ch1 = lds + C;
    float* s0 = lds + 2 * C;
    float* s1 = s0 + R * width;
    const long long r0 = (long long)chunk * p.rows;
    const int n = (int)(p.HW - r0 < p.rows ? p.HW - r0 : p.rows);
    const int col = threadIdx.x % pc, rl = threadIdx.x / pc;
    float* o = p.chan + ((long long)b * p.nchunk + chunk) * 2 * C;
    for (int c0 = 0; c0 < cols; c0 += pc) {
        const int c = c0 + col;
        if (rl < R && c < cols) {
            float mean[VEC], rstd[VEC], gm[VEC], bt[VEC], a[VEC], q[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int ch = c * VEC + e, g = ch / cg;
                mean[e] = p.mean[(long long)b * p.G + g];
                rstd[e] = p.rstd[(long long)b * p.G + g];
                gm[e] = p.gamma[ch];
                bt[e] = p.beta[ch];
                a[e] = q[e] = 0.f;
            }
            const T* x = (const T*)p.x + b * p.x_b + r0 * p.x_row + (long long)c * VEC;
            const T* dy = (const T*)p.dy + b * p.dy_b + r0 * p.dy_row + (long long)c * VEC;
#pragma unroll 2
            for (int r = rl; r < n; r += R) {
                float v[VEC], d[VEC];
                load_vec<T, VEC>(x + r * p.x_row, v);
                load_vec<T, VEC>(dy + r * p.dy_row, d);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float xh = (v[e] - mean[e]) * rstd[e];
                    const float dz = dz_of(d[e], xh * gm[e] + bt[e], p.act);
                    a[e] += dz;
                    q[e] += dz * xh;
                }
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                s0[rl * width + col * VEC + e] = a[e];
                s1[rl * width + col * VEC + e] = q[e];
            }
        }
        fold_rows<VEC>(s0, s1, R, width);
        const int w = (cols - c0 < pc ? cols - c0 : pc) * VEC;
        for (int i = threadIdx.x; i < w; i += NT) {
            const float gm = p.gamma[c0 * VEC + i];
            o[c0 * VEC + i] = s0[i];
            o[C + c0 * VEC + i] = s1[i];
            ch0[c0 * VEC + i] = gm * s0[i];
            ch1[c0 * VEC + i] = gm * s1[i];
        }
        __syncthreads();
    }
    const int lanes = lanes_per(p.G), sub = threadIdx.x % lanes, stride = NT / lanes;
    for (int g0 = 0; g0 < p.G; g0 += stride) {
        const int g = min(g0 + (int)threadIdx.x / lanes, p.G - 1);
        float a = 0.f, q = 0.f;
        for (int c = sub; c < cg; c += lanes) {
            a += ch0[g * cg + c];
            q += ch1[g * cg + c];
        }
        a = lanes_sum(a, lanes);
        q = lanes_sum(q, lanes);
        if (sub == 0) *reinterpret_cast<f32x2*>(p.part + (((long long)b * p.nchunk + chunk) * p.G + g) * 2) = f32x2{a, q};
    }
}

// ---- backward, launch 2: the group means from the chunks' sums, then dx of one chunk.  The first p.tail blocks (they run longest)
// sum dgamma and dbeta instead, 64 channels each: 64 lanes x 4 runs of the B * nchunk chunk sums, joined in order.
template <typename T, int VEC> __global__ void __launch_bounds__(NT) k_gna_bwd_dx(NormArgs p, int tail) {
    extern __shared__ float lds[];
    const int C = p.C, cols = C / VEC, cg = C / p.G;
    if ((int)blockIdx.x < tail) {
        const int c = blockIdx.x * 64 + (threadIdx.x & 63), run = threadIdx.x >> 6;
        const long long all = (long long)p.B * p.nchunk, per = (all + 3) / 4, i0 = run * per, i1 = i0 + per < all ? i0 + per : all;
        float a = 0.f, q = 0.f;
        if (c < C) {
            const float* o = p.chan + c;
#pragma unroll 8
            for (long long i = i0; i < i1; ++i) {
                a += o[i * 2 * C];
                q += o[i * 2 * C + C];
            }
        }
        lds[threadIdx.x] = a;
        lds[NT + threadIdx.x] = q;
        __syncthreads();
        if (run == 0 && c < C) {
            p.dbeta[c] = (lds[threadIdx.x] + lds[64 + threadIdx.x]) + (lds[128 + threadIdx.x] + lds[192 + threadIdx.x]);
            p.dgamma[c] = (lds[NT + threadIdx.x] + lds[NT + 64 + threadIdx.x]) + (lds[NT + 128 + threadIdx.x] + lds[NT + 192 + threadIdx.x]);
        }
        return;
    }
    const int id = blockIdx.x - tail, chunk = id % p.nchunk, b = id / p.nchunk;
    float* ga = lds;                      // [G]
    float* gq = lds + p.G;
    const int lanes = lanes_per(p.G), sub = threadIdx.x % lanes, stride = NT / lanes;
    const float inv = 1.0f / ((float)p.HW * (float)cg);
    for (int g0 = 0; g0 < p.G; g0 += stride) {
        const int g = min(g0 + (int)threadIdx.x / lanes, p.G - 1);
        const f32x2* o = reinterpret_cast<const f32x2*>(p.part) + (long long)b * p.nchunk * p.G + g;
        float a = 0.f, q = 0.f;
#pragma unroll 4
        for (int i = sub; i < p.nchunk; i += lanes) {
            const f32x2 t = o[(long long)i * p.G];
            a += t[0];
            q += t[1];
        }
        a = lanes_sum(a, lanes);
        q = lanes_sum(q, lanes);
        if (sub == 0) {
            ga[g] = a * inv;
            gq[g] = q * inv;
        }
    }
    __syncthreads();
    const int pc = cols < NT ? cols : NT, R = NT / pc;
    const long long r0 = (long long)chunk * p.rows;
    const int n = (int)(p.HW - r0 < p.rows ? p.HW - r0 : p.rows);
    const int col = threadIdx.x % pc, rl = threadIdx.x / pc;
    if (rl >= R) return;
    for (int c = col; c < cols; c += pc) {
        float mean[VEC], rstd[VEC], gm[VEC], bt[VEC], ka[VEC], kb[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int ch = c * VEC + e, g = ch / cg;
            const long long bg = (long long)b * p.G + g;
            mean[e] = p.mean[bg];
            rstd[e] = p.rstd[bg];
            gm[e] = p.gamma[ch];
            bt[e] = p.beta[ch];
            ka[e] = ga[g];
            kb[e] = gq[g];
        }
        const T* x = (const T*)p.x + b * p.x_b + r0 * p.x_row + (long long)c * VEC;
        const T* dy = (const T*)p.dy + b * p.dy_b + r0 * p.dy_row + (long long)c * VEC;
        T* dx = (T*)p.out + ((long long)b * p.HW + r0) * C + (long long)c * VEC;
#pragma unroll 2
        for (int r = rl; r < n; r += R) {
            float v[VEC], d[VEC];
            load_vec<T, VEC>(x + r * p.x_row, v);
            load_vec<T, VEC>(dy + r * p.dy_row, d);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float xh = (v[e] - mean[e]) * rstd[e];
                const float dz = dz_of(d[e], xh * gm[e] + bt[e], p.act);
                v[e] = rstd[e] * (gm[e] * dz - ka[e] - xh * kb[e]);
            }
            store_vec<T, VEC>(dx + (long long)r * C, v);
        }
    }
}

bool aligned16(const void* p, long long s0, long long s1, int esize) {
    return ((uintptr_t)p % 16) == 0 && (s0 * esize) % 16 == 0 && (s1 * esize) % 16 == 0;
}

int check_args(const char* name, const void* x, long long x_b, long long x_row, int dtype, int B, long long HW, int C, int G, const float* gamma,
               const float* beta, int act, int rows) {
    VS_REQUIRE(x && gamma && beta, "%s: null operand", name);
    VS_REQUIRE(dtype >= 0 && dtype <= 2, "%s: dtype %d (0 fp32, 1 fp16, 2 bf16)", name, dtype);
    VS_REQUIRE(B >= 1 && B <= 65535 && HW >= 1 && C >= 1 && C <= 8192 && G >= 1 && C % G == 0, "%s: B=%d HW=%lld C=%d G=%d", name, B, HW, C, G);
    VS_REQUIRE(act == 0 || act == 1, "%s: act %d (0 none, 1 SiLU)", name, act);
    VS_REQUIRE(rows >= 1 && (HW + rows - 1) / rows <= (1 << 20), "%s: rows_per_chunk=%d", name, rows);
    VS_REQUIRE(x_row >= C && x_b >= 0, "%s: row stride %lld below C=%d", name, x_row, C);
    return VS_OK;
}

// CALL(T, VEC): 16-byte accesses where every operand allows them, single values otherwise (28 x 4096 x 320 fp16: 51 us, one element off alignment 130)
#define GNA_DISPATCH(dtype, wide, CALL)                      \
    do {                                                     \
        if ((dtype) == 0) {                                  \
            if (wide) { CALL(float, 4); } else { CALL(float, 1); }        \
        } else if ((dtype) == 1) {                           \
            if (wide) { CALL(_Float16, 8); } else { CALL(_Float16, 1); }  \
        } else {                                             \
            if (wide) { CALL(__bf16, 8); } else { CALL(__bf16, 1); }      \
        }                                                    \
    } while (0)

size_t fold_floats(int C, int VEC) {
    const int cols = C / VEC, pc = cols < NT ? cols : NT, R = NT / pc;
    return (size_t)2 * R * pc * VEC;
}

// More than 64 KB of LDS has to be asked for; the widest maps (C = 8192) need 80 KB
template <void (*K)(NormArgs)> int allow_lds() {
    static VsOncePerDevice once;
    if (once.needs()) {
        hipError_t e = hipFuncSetAttribute((const void*)K, hipFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024);
        if (e != hipSuccess) VS_FAIL(VS_ERR_HIP, "groupnorm_act: %s", hipGetErrorString(e));
        once.mark();
    }
    return VS_OK;
}

}  // namespace

extern "C" {

int vidseg_groupnorm_act_fwd(const void* x, long long x_batch_stride, long long x_row_stride, int dtype, int B, long long HW, int C, int G,
                             const float* gamma, const float* beta, float eps, int act, int rows_per_chunk, void* y, float* mean, float* rstd,
                             float* scratch, long long scratch_floats, hipStream_t s) {
    const int rc = check_args("groupnorm_act", x, x_batch_stride, x_row_stride, dtype, B, HW, C, G, gamma, beta, act, rows_per_chunk);
    if (rc) return rc;
    VS_REQUIRE(y && scratch && (!mean == !rstd), "groupnorm_act: null output or scratch");
    NormArgs p{};
    p.x = x; p.x_b = x_batch_stride; p.x_row = x_row_stride; p.HW = HW; p.B = B; p.C = C; p.G = G; p.rows = rows_per_chunk;
    p.nchunk = (int)((HW + rows_per_chunk - 1) / rows_per_chunk);
    p.down = eps >= 0x1p-60f ? 0x1p-32f : 1.0f;
    p.act = act; p.eps = eps; p.gamma = gamma; p.beta = beta; p.out = y; p.mean = mean; p.rstd = rstd; p.part = scratch;
    VS_REQUIRE((long long)B * p.nchunk * G * 2 <= scratch_floats, "groupnorm_act: scratch of %lld floats, needs %lld", scratch_floats,
               (long long)B * p.nchunk * G * 2);
    const int es = dtype == 0 ? 4 : 2, vec = 16 / es;
    const bool wide = C % vec == 0 && aligned16(x, x_batch_stride, x_row_stride, es) && aligned16(y, 0, 0, es);
    const dim3 grid(p.nchunk, B);
    const size_t l1 = (2 * (size_t)C + fold_floats(C, wide ? vec : 1)) * 4, l2 = 2 * (size_t)G * 4;
#define CALL(T, V)                                                       \
    if (int rc2 = allow_lds<k_gna_stats<T, V>>()) return rc2; \
    hipLaunchKernelGGL((k_gna_stats<T, V>), grid, dim3(NT), l1, s, p);   \
    hipLaunchKernelGGL((k_gna_apply<T, V>), grid, dim3(NT), l2, s, p)
    GNA_DISPATCH(dtype, wide, CALL);
#undef CALL
    VS_CHECK_LAUNCH("groupnorm_act");
    return VS_OK;
}

int vidseg_groupnorm_act_bwd(const void* dy, long long dy_batch_stride, long long dy_row_stride, const void* x, long long x_batch_stride,
                             long long x_row_stride, int dtype, int B, long long HW, int C, int G, const float* gamma, const float* beta,
                             const float* mean, const float* rstd, int act, int rows_per_chunk, void* dx, float* dgamma, float* dbeta,
                             float* scratch, long long scratch_floats, hipStream_t s) {
    const int rc = check_args("groupnorm_act_bwd", x, x_batch_stride, x_row_stride, dtype, B, HW, C, G, gamma, beta, act, rows_per_chunk);
    if (rc) return rc;
    VS_REQUIRE(dy && mean && rstd && dx && dgamma && dbeta && scratch, "groupnorm_act_bwd: null operand");
    VS_REQUIRE(dy_row_stride >= C && dy_batch_stride >= 0, "groupnorm_act_bwd: gradient row stride %lld below C=%d", dy_row_stride, C);
    NormArgs p{};
    p.x = x; p.x_b = x_batch_stride; p.x_row = x_row_stride; p.dy = dy; p.dy_b = dy_batch_stride; p.dy_row = dy_row_stride;
    p.HW = HW; p.B = B; p.C = C; p.G = G; p.rows = rows_per_chunk;
    p.nchunk = (int)((HW + rows_per_chunk - 1) / rows_per_chunk);
    p.act = act; p.gamma = gamma; p.beta = beta; p.out = dx; p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd);
    p.part = scratch;
    p.chan = scratch + 2ll * B * p.nchunk * G;
    p.dgamma = dgamma; p.dbeta = dbeta;
    const long long need = 2ll * B * p.nchunk * ((long long)C + G), tail = (C + 63) / 64;
    VS_REQUIRE(need <= scratch_floats, "groupnorm_act_bwd: scratch of %lld floats, needs %lld", scratch_floats, need);
    const int es = dtype == 0 ? 4 : 2, vec = 16 / es;
    const bool wide = C % vec == 0 && aligned16(x, x_batch_stride, x_row_stride, es) && aligned16(dy, dy_batch_stride, dy_row_stride, es) &&
                      aligned16(dx, 0, 0, es);
    VS_REQUIRE((long long)p.nchunk * B + tail < (1ll << 24), "groupnorm_act_bwd: B=%d HW=%lld are too many chunks of %d rows", B, HW, rows_per_chunk);
    const dim3 grid(p.nchunk, B), grid2((unsigned)(p.nchunk * (long long)B + tail));
    const size_t l1 = (2 * (size_t)C + fold_floats(C, wide ? vec : 1)) * 4, l2 = (size_t)(2 * G > 2 * NT ? 2 * G : 2 * NT) * 4;
#define CALL(T, V)                                                        \
    if (int rc2 = allow_lds<k_gna_bwd_sums<T, V>>()) return rc2; \
    hipLaunchKernelGGL((k_gna_bwd_sums<T, V>), grid, dim3(NT), l1, s, p); \
    hipLaunchKernelGGL((k_gna_bwd_dx<T, V>), grid2, dim3(NT), l2, s, p, (int)tail)
    GNA_DISPATCH(dtype, wide, CALL);
#undef CALL
    VS_CHECK_LAUNCH("groupnorm_act_bwd");
    return VS_OK;
}

}  // extern "C"
