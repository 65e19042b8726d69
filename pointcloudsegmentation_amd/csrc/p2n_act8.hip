// Training layers that keep their input for the backward pass in 8 bits (gfx950).
//     h = W . a + b,   a = relu(norm(x))  or  a = x          x (B, K, L), W (N, K), h (B, N, L)
// norm is BatchNorm over the B*L points of a channel (reference point2net.py:9-34 in train() mode): mean and biased variance
// from sums in 64 bits, mu and r = 1/sqrt(var + eps) kept as float32, u = fl(fl(x - mu) * r), y = gamma*u + beta.
// Kept instead of x: the codes of u (of x without a norm) by the 8-bit rule of p2n_q8.h, one scale for 128 consecutive points of a
// (cloud, channel) row, and one bit [y > 0] for each value, so the ReLU's decisions stay exact: 1.16 bytes a value for 4.
// A NaN counts as above zero, so it goes on into everything that its value enters, on the way back too.
// The backward pass works from uh = s*q and ah = [y > 0] * max(gamma*uh + beta, 0):
//     dW = g . ah^T   db = sum g   da = W^T . g   dy = [y > 0] * da   dbeta = sum dy   dgamma = sum dy*uh
//     dx = gamma*r*(dy - dbeta/P - uh*dgamma/P),  P = B*L   (frozen statistics: gamma*r*dy;  without a norm: da)
// The reference keeps float32 activations (train.py:124-131 under autograd); the formulas above are the specification.
//
// Products of float32 operands run on the bf16 matrix cores: each operand is the exact sum of three bf16 parts (24 bits),
// and of the nine part products the six that reach 2^-16 of the largest are added in float32 -- float32 accuracy at
// 1/6 of the bf16 rate, against 1/16 for the float32 instruction.
#include "p2n_q8.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
#define MFMAB(a, b, c) __builtin_amdgcn_mfma_f32_32x32x16_bf16((a), (b), (c), 0, 0, 0)
#define ACT8_MAX_C 1024
#define ACT8_GROUP 128

#define TRY(expr)                  \
    do {                           \
        const int rc_ = (expr);    \
        if (rc_) return rc_;       \
    } while (0)

// ---------------------------------------------------------------- what is kept
// codes (B, C, 128 NB) | scales (B, C, NB) | bits (B, C, 4 NB) 32-bit words | mu[C], r[C];  NB = ceil(L / 128); codes and
// bits behind the last point are zero
struct Act8Kept {
    long NB;
    size_t scale, bits, stat, total;
};

static Act8Kept act8_kept(int B, int C, long L, int norm) {
    Act8Kept k;
    k.NB = (L + ACT8_GROUP - 1) / ACT8_GROUP;
    const size_t groups = (size_t)B * C * k.NB;
    k.scale = groups * ACT8_GROUP;
    k.bits = k.scale + ((groups * 4 + 255) & ~(size_t)255);
    k.stat = k.bits + (norm ? (groups * 16 + 255) & ~(size_t)255 : 0);
    k.total = k.stat + (norm ? ((size_t)C * 8 + 255) & ~(size_t)255 : 0);
    return k;
}

__device__ __forceinline__ float act8_relu(float y) { return y <= 0.f ? 0.f : y; }   // a NaN stays

// ---------------------------------------------------------------- BatchNorm statistics
// grid (C, S): sums of (x - pivot) and its square over a slice of the (cloud, block) list, in 64 bits, pivot = x[0][c][0]
__global__ __launch_bounds__(256) void p2n_act8_stats_kernel(const float *__restrict__ x, int B, int C, long L, long blocks, long per, double *__restrict__ part) {
    __shared__ double sh[8];
    const int c = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long NB = (L + 1023) / 1024;                      // a block: 1024 columns of a cloud
    const float pivot = x[(long)c * L];
    double u = 0.0, v = 0.0;
    const long b0 = (long)blockIdx.y * per, b1 = b0 + per < blocks ? b0 + per : blocks;
    for (long i = b0; i < b1; ++i) {
        const long b = i / NB, l0 = (i % NB) * 1024;
        const float *row = x + (b * C + c) * L;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const long l = l0 + 256 * j + threadIdx.x;
            if (l < L) {
                const double d = (double)row[l] - (double)pivot;
                u += d;
                v += d * d;
            }
        }
    }
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        u += __shfl_xor(u, m);
        v += __shfl_xor(v, m);
    }
    if (lane == 0) { sh[wave] = u; sh[4 + wave] = v; }
    __syncthreads();
    if (threadIdx.x == 0) {
        part[((long)c * gridDim.y + blockIdx.y) * 2] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
        part[((long)c * gridDim.y + blockIdx.y) * 2 + 1] = (sh[4] + sh[5]) + (sh[6] + sh[7]);
    }
}

// mu, r kept as float32; tab = {mu, gamma*r, beta} for the forward loader, zero behind the last channel.  frozen: from the
// running statistics.  One thread a channel.
__global__ void p2n_act8_norm_kernel(const double *__restrict__ part, int S, const float *__restrict__ x, int C, int Cpad, long L, double P,
                                     const float *__restrict__ gamma, const float *__restrict__ beta, float *__restrict__ rmean,
                                     float *__restrict__ rvar, double momentum, double eps, int frozen, float *__restrict__ stat, float *__restrict__ tab) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= Cpad) return;
    if (c >= C) {
        tab[c] = tab[Cpad + c] = tab[2 * Cpad + c] = 0.f;
        return;
    }
    double mean, var;
    if (frozen) {
        mean = rmean[c];
        var = rvar[c];
    } else {
        double u = 0.0, v = 0.0;
        for (int s = 0; s < S; ++s) { u += part[((long)c * S + s) * 2]; v += part[((long)c * S + s) * 2 + 1]; }
        const double d = u / P;
        mean = (double)x[(long)c * L] + d;
        var = v / P - d * d;
        if (var < 0.0) var = 0.0;
        if (rmean) {
            rmean[c] = (float)((1.0 - momentum) * rmean[c] + momentum * mean);
            rvar[c] = (float)((1.0 - momentum) * rvar[c] + momentum * var * (P / (P - 1.0)));
        }
    }
    const float mu = (float)mean, r = (float)(1.0 / sqrt(var + eps));
    stat[c] = mu;
    stat[C + c] = r;
    tab[c] = mu;
    tab[Cpad + c] = gamma[c] * r;
    tab[2 * Cpad + c] = beta[c];
}

// ---------------------------------------------------------------- codes
// one wave per group of 128 points: u, its scale, codes, the ReLU's bits
template <bool NORM>
__global__ __launch_bounds__(256) void p2n_act8_pack_kernel(const float *__restrict__ x, long groups, int C, long L, long NB, const float *__restrict__ stat,
                                                            const float *__restrict__ gamma, const float *__restrict__ beta, signed char *__restrict__ codes,
                                                            float *__restrict__ scale, unsigned *__restrict__ bits) {
    const int lane = threadIdx.x & 63;
    const long grp = (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (grp >= groups) return;
    const long row = grp / NB, l0 = (grp % NB) * ACT8_GROUP;      // row = cloud * C + channel
    const int c = (int)(row % C);
    const float *p = x + row * L + l0;
    const bool ok0 = l0 + lane < L, ok1 = l0 + 64 + lane < L;
    float v0 = ok0 ? p[lane] : 0.f, v1 = ok1 ? p[64 + lane] : 0.f;
    if (NORM) {
        const float mu = stat[c], r = stat[C + c], ga = gamma[c], be = beta[c];
        v0 = ok0 ? (v0 - mu) * r : 0.f;
        v1 = ok1 ? (v1 - mu) * r : 0.f;
        const unsigned long long m0 = __ballot(ok0 && !(fmaf(ga, v0, be) <= 0.f)), m1 = __ballot(ok1 && !(fmaf(ga, v1, be) <= 0.f));
        if (lane < 4) bits[grp * 4 + lane] = (unsigned)((lane < 2 ? m0 : m1) >> (32 * (lane & 1)));
    }
    unsigned am = p2n_absbits(v0), o = p2n_absbits(v1);
    am = o > am ? o : am;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        o = (unsigned)__shfl_xor((int)am, m);
        am = o > am ? o : am;
    }
    const float s = p2n_q8_scale(am);
    const P2nQ8 Q = p2n_q8_make(s);
    const bool bad = !(s == s);
    if (lane == 0) scale[grp] = s;
    codes[grp * ACT8_GROUP + lane] = bad ? 0 : (signed char)p2n_q8_decide(v0, Q);
    codes[grp * ACT8_GROUP + 64 + lane] = bad ? 0 : (signed char)p2n_q8_decide(v1, Q);
}

// ---------------------------------------------------------------- weight image of a product
// three-way split w = h + m + l: fragment (ks * CTP + ct) * 3 + part, 1 KiB: lane holds part(M[32ct + (lane&31)][16ks + 8(lane>>5) + i]),
// i < 8; M = W (rows N) or W^T (rows K); zero outside.  CTP = channel tiles rounded up to what a workgroup makes.
__global__ __launch_bounds__(256) void p2n_act8_split_kernel(const float *__restrict__ W, int rows, int cols, int trans, int CTP, int KS, __bf16 *__restrict__ img) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;          // (fragment without part, lane)
    const int lane = (int)(i & 63);
    const long f = i >> 6;
    if (f >= (long)CTP * KS) return;
    const int ct = (int)(f % CTP), ks = (int)(f / CTP);
    const int row = 32 * ct + (lane & 31), k0 = 16 * ks + 8 * (lane >> 5);
    bf16x8 h, m, l;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int k = k0 + j;
        const float v = row < rows && k < cols ? (trans ? W[(long)k * rows + row] : W[(long)row * cols + k]) : 0.f;
        h[j] = (__bf16)v;
        const float r = v - (float)h[j];
        m[j] = (__bf16)r;
        l[j] = (__bf16)(r - (float)m[j]);
    }
    bf16x8 *d = reinterpret_cast<bf16x8 *>(img) + f * 3 * 64 + lane;
    d[0] = h; d[64] = m; d[128] = l;
}

// ---------------------------------------------------------------- products over points
// D = M . X, lane = point, registers = channels.  A workgroup takes 128 points (one group of a cloud), a wave 32 of them and all of
// CT*32 output channels; the weight fragments pass through LDS (double buffer, LDS-DMA), X through registers.
struct Act8Gemm {
    const float *x;        // (B, K, L)
    const __bf16 *img;
    const float *tab;      // ACT8_NORM: {mu, gamma*r, beta}[Kpad]
    const float *bias;     // NULL, or one a row
    float *out;            // (B, rows, L)
    const signed char *codes;   // ACT8_DY: what was kept, rows channels
    const float *scale;
    const unsigned *bits;
    float *part;           // ACT8_DY: {sum dy, sum dy*uh}[rows][2][gridDim.x]
    long L, NB;
    int K, Kpad, KS, CTP, rows;
};
enum { ACT8_PLAIN = 0, ACT8_NORM = 1 };     // operand
enum { ACT8_OUT = 0, ACT8_DY = 1 };         // epilogue

typedef __attribute__((address_space(3))) void act8_lds_t;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t act8_rsrc(const void *base, long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, (int)(bytes < 0xFFFFFFFFL ? bytes : 0xFFFFFFFFL), 0x00020000);
}

__device__ __forceinline__ f32x16 act8_mma6(f32x16 acc, bf16x8 ah, bf16x8 am, bf16x8 al, bf16x8 bh, bf16x8 bm, bf16x8 bl) {
    acc = MFMAB(al, bh, acc);      // the small ones first
    acc = MFMAB(ah, bl, acc);
    acc = MFMAB(am, bm, acc);
    acc = MFMAB(am, bh, acc);
    acc = MFMAB(ah, bm, acc);
    return MFMAB(ah, bh, acc);
}

__device__ __forceinline__ void act8_split(const float (&v)[8], bf16x8 &h, bf16x8 &m, bf16x8 &l) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        h[i] = (__bf16)v[i];
        const float r = v[i] - (float)h[i];
        m[i] = (__bf16)r;
        l[i] = (__bf16)(r - (float)m[i]);
    }
}

// sums of 16 registers over the 32 lanes of a half, as p2n_tile_half_max: lane i of a 16-lane row ends with register i's sum
template <int N, int CTRL>
__device__ __forceinline__ void act8_halve_sum(float (&m)[16], bool upper) {
#pragma unroll
    for (int q = 0; q < N; ++q) {
        const float keep = upper ? m[2 * q + 1] : m[2 * q], give = upper ? m[2 * q] : m[2 * q + 1];
        m[q] = keep + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(give), CTRL, 0xF, 0xF, true));
    }
}
__device__ __forceinline__ float act8_half_sum(float (&m)[16], int lane) {
    act8_halve_sum<8, 0xB1>(m, lane & 1);
    act8_halve_sum<4, 0x4E>(m, lane & 2);
    act8_halve_sum<2, 0x124>(m, lane & 4);
    act8_halve_sum<1, 0x128>(m, lane & 8);
    return m[0] + __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(m[0]), 0x401F));
}

template <int IN, int EPI, int CT>
__global__ __launch_bounds__(256, CT <= 4 ? 3 : 2) void p2n_act8_gemm_kernel(Act8Gemm A) {
    constexpr int CKS = CT >= 4 ? 1 : 4 / CT;       // k-steps of 16 in a chunk: 12 or 24 fragments, a multiple of the four waves
    constexpr int F = CKS * CT * 3;
    __shared__ __attribute__((aligned(16))) char wbuf[2][F * 1024];
    __shared__ __attribute__((aligned(16))) float tab[IN == ACT8_NORM ? 3 * ACT8_MAX_C : 4];
    __shared__ float red[EPI == ACT8_DY ? 4 * 2 * 32 * CT : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int p = lane & 31, h = lane >> 5;
    const long b = blockIdx.x / A.NB, nb = blockIdx.x % A.NB, l = nb * ACT8_GROUP + 32 * wave + p;
    const bool valid = l < A.L;
    const int ct0 = blockIdx.y * CT;                 // first channel tile of this workgroup
    const int nchunk = A.KS / CKS;
    const float *xb = A.x + b * A.K * A.L;
    const unsigned off = (unsigned)((8 * h * A.L + (valid ? l : A.L - 1)) * 4);
    if (IN == ACT8_NORM)
        for (int i = threadIdx.x; i < 3 * A.Kpad; i += 256) tab[i] = A.tab[i];

    auto stage = [&](int c) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t rs = act8_rsrc(A.img, (long)A.CTP * A.KS * 3072);
#pragma unroll
        for (int i = 0; i < F / 4; ++i) {
            const int f = wave * (F / 4) + i;        // fragment of the chunk: k-step f / (3 CT), the rest in image order
            const int ks = c * CKS + f / (3 * CT);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (act8_lds_t *)(wbuf[c & 1] + f * 1024), 16, lane * 16,
                                                     ((ks * A.CTP + ct0) * 3 + f % (3 * CT)) * 1024, 0, 0);
        }
    };
    float raw[CKS][8];
    auto fetch = [&](int c) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < CKS; ++s) {
            const int k0 = 16 * (c * CKS + s);
            const long left = (long)(A.K - k0) * A.L * 4;
            const __amdgpu_buffer_rsrc_t rs = act8_rsrc(xb + (long)k0 * A.L, left > 0 ? left : 0);   // rows past the last read as zero
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[s][i] = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, off + (unsigned)(i * A.L * 4), 0, 0));
        }
    };
    f32x16 acc[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[ct][e] = 0.f;
    stage(0);
    fetch(0);
#pragma unroll 1
    for (int c = 0; c < nchunk; ++c) {
        p2n_dma_barrier();                            // chunk c is in LDS, this wave's rows of it in registers
        bf16x8 xh[CKS], xm[CKS], xl[CKS];
#pragma unroll
        for (int s = 0; s < CKS; ++s) {
            if (IN == ACT8_NORM) {
                const int k = 16 * (c * CKS + s) + 8 * h;
#pragma unroll
                for (int i = 0; i < 8; ++i) raw[s][i] = act8_relu(fmaf(raw[s][i] - tab[k + i], tab[A.Kpad + k + i], tab[2 * A.Kpad + k + i]));
            }
            act8_split(raw[s], xh[s], xm[s], xl[s]);
        }
        if (c + 1 < nchunk) {
            stage(c + 1);
            fetch(c + 1);
        }
#pragma unroll
        for (int s = 0; s < CKS; ++s)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const bf16x8 *w = reinterpret_cast<const bf16x8 *>(wbuf[c & 1] + (s * CT + ct) * 3072) + lane;
                acc[ct] = act8_mma6(acc[ct], w[0], w[64], w[128], xh[s], xm[s], xl[s]);
            }
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        const int r0 = 32 * (ct0 + ct);
        if (r0 >= A.rows) continue;
        const __amdgpu_buffer_rsrc_t ro = act8_rsrc(A.out + (b * A.rows + r0) * A.L, (long)(A.rows - r0) * A.L * 4);
        const unsigned oo = (unsigned)((4 * h * A.L + l) * 4);
        if (EPI == ACT8_DY) {
            float s1[16], s2[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int row = r0 + 8 * (e >> 2) + 4 * h + (e & 3);
                const long grp = (b * A.rows + (row < A.rows ? row : A.rows - 1)) * A.NB + nb;
                const bool on = row < A.rows && (A.bits[grp * 4 + wave] >> p & 1);
                const float uh = (float)A.codes[grp * ACT8_GROUP + 32 * wave + p] * A.scale[grp];
                const float dy = on ? acc[ct][e] : 0.f;
                acc[ct][e] = dy;
                s1[e] = dy;
                s2[e] = on ? dy * uh : 0.f;
            }
            const float t1 = act8_half_sum(s1, lane), t2 = act8_half_sum(s2, lane);
            const int i = lane & 15, c = 32 * ct + 8 * (i >> 2) + 4 * h + (i & 3);
            if (!(lane & 16)) {
                red[(wave * 2) * 32 * CT + c] = t1;
                red[(wave * 2 + 1) * 32 * CT + c] = t2;
            }
        }
        if (valid) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float v = acc[ct][e];
                if (EPI == ACT8_OUT && A.bias) {
                    const int row = r0 + 8 * (e >> 2) + 4 * h + (e & 3);
                    v += A.bias[row < A.rows ? row : A.rows - 1];
                }
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(v), ro, oo + (unsigned)((8 * (e >> 2) + (e & 3)) * A.L * 4), 0, 0);
            }
        }
    }
    if (EPI == ACT8_DY) {
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * 32 * CT; i += 256) {
            const int which = i / (32 * CT), c = i % (32 * CT), row = 32 * ct0 + c;
            if (row >= A.rows) continue;
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) s += red[(w * 2 + which) * 32 * CT + c];
            A.part[((long)row * 2 + which) * gridDim.x + blockIdx.x] = s;
        }
    }
}

// ---------------------------------------------------------------- the rest of the norm's backward
// sums of a row's partials, in 64 bits and in order: dbeta, dgamma, and {gamma*r, m1, m2} for dx
__global__ __launch_bounds__(256) void p2n_act8_sums_kernel(const float *__restrict__ part, long n, int C, double P, const float *__restrict__ gamma,
                                                            const float *__restrict__ stat, int frozen, float *__restrict__ dgamma, float *__restrict__ dbeta,
                                                            float *__restrict__ tab) {
    __shared__ double sh[8];
    const int c = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double u = 0.0, v = 0.0;
    for (long i = threadIdx.x; i < n; i += 256) {
        u += part[((long)c * 2) * n + i];
        v += part[((long)c * 2 + 1) * n + i];
    }
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        u += __shfl_xor(u, m);
        v += __shfl_xor(v, m);
    }
    if (lane == 0) { sh[wave] = u; sh[4 + wave] = v; }
    __syncthreads();
    if (threadIdx.x == 0) {
        u = (sh[0] + sh[1]) + (sh[2] + sh[3]);
        v = (sh[4] + sh[5]) + (sh[6] + sh[7]);
        if (dbeta) dbeta[c] = (float)u;
        if (dgamma) dgamma[c] = (float)v;
        tab[c] = gamma[c] * stat[C + c];
        tab[C + c] = frozen ? 0.f : (float)(u / P);
        tab[2 * C + c] = frozen ? 0.f : (float)(v / P);
    }
}

// dx = gamma*r*(dy - m1 - uh*m2), in place; one wave per group
__global__ __launch_bounds__(256) void p2n_act8_dx_kernel(float *__restrict__ dy, long groups, int C, long L, long NB, const float *__restrict__ tab,
                                                          const signed char *__restrict__ codes, const float *__restrict__ scale) {
    const int lane = threadIdx.x & 63;
    const long grp = (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (grp >= groups) return;
    const long row = grp / NB, l0 = (grp % NB) * ACT8_GROUP;
    const int c = (int)(row % C);
    const float a = tab[c], m1 = tab[C + c], m2 = tab[2 * C + c], s = scale[grp];
    float *d = dy + row * L + l0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int i = 64 * j + lane;
        if (l0 + i < L) d[i] = a * (d[i] - m1 - (float)codes[grp * ACT8_GROUP + i] * s * m2);
    }
}

// ---------------------------------------------------------------- weight gradient
// dW[n][k] = sum over points g[n] * ah[k]: both operands are rows of consecutive points.  A workgroup makes 128 x 128 of dW over a
// slice of the points, 32 at a time, split into three bf16 parts on the way to LDS; slices are added by a second kernel, in order.
struct Act8Wgrad {
    const float *g;        // (B, N, L)
    const signed char *codes;   // (B, K, 128 NB)
    const float *scale;
    const unsigned *bits;  // NULL: a = uh
    const float *gamma, *beta;
    float *part;           // [slices][N][K]
    float *dbpart;         // [slices][N]
    long L, NB, steps, per;   // steps of 32 points in all, per slice
    int N, K;
};
#define AW_LD 40                            // bf16 elements per parked row of 32 points (80 bytes)
#define AW_TILE (128 * AW_LD)

__global__ __launch_bounds__(256, 2) void p2n_act8_wgrad_kernel(Act8Wgrad A) {
    __shared__ __attribute__((aligned(16))) __bf16 sa[3 * AW_TILE], sb[3 * AW_TILE];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int r = lane & 31, h = lane >> 5, wr = wave >> 1, wc = wave & 1;
    const int ntc = (A.K + 127) / 128;
    const int n0 = (blockIdx.x / ntc) * 128, k0 = (blockIdx.x % ntc) * 128;
    const long s0 = (long)blockIdx.y * A.per, s1 = s0 + A.per < A.steps ? s0 + A.per : A.steps;
    const long spc = 4 * A.NB;              // steps of a cloud
    // staging: a thread takes 8 consecutive points of rows t/4 and t/4 + 64 of either operand
    const int seg = (t & 3) * 8, srow = t >> 2;
    float ga[2], be[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int k = k0 + srow + 64 * i;
        ga[i] = A.bits && k < A.K ? A.gamma[k] : 1.f;
        be[i] = A.bits && k < A.K ? A.beta[k] : 0.f;
    }
    float va[2][8], sc[2], db[2] = {0.f, 0.f};
    unsigned long long qb[2];
    unsigned mb[2];
    auto fetch = [&](long s) __attribute__((always_inline)) {
        const long b = s / spc, l0 = (s % spc) * 32, l = l0 + seg;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int n = n0 + srow + 64 * i, k = k0 + srow + 64 * i;
            const float *q = A.g + (b * A.N + (n < A.N ? n : A.N - 1)) * A.L;
#pragma unroll
            for (int j = 0; j < 8; ++j) va[i][j] = n < A.N && l + j < A.L ? q[l + j] : 0.f;
            const long grp = (b * A.K + (k < A.K ? k : A.K - 1)) * A.NB + (l0 >> 7);
            qb[i] = *reinterpret_cast<const unsigned long long *>(A.codes + grp * ACT8_GROUP + (l0 & 127) + seg);
            sc[i] = k < A.K ? A.scale[grp] : 0.f;
            mb[i] = k < A.K ? (A.bits ? A.bits[grp * 4 + ((l0 >> 5) & 3)] >> seg : 0xFFu) : 0u;
        }
    };
    auto park = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            bf16x8 xh, xm, xl;
            act8_split(va[i], xh, xm, xl);
            __bf16 *d = sa + (srow + 64 * i) * AW_LD + seg;
            *reinterpret_cast<bf16x8 *>(d) = xh;
            *reinterpret_cast<bf16x8 *>(d + AW_TILE) = xm;
            *reinterpret_cast<bf16x8 *>(d + 2 * AW_TILE) = xl;
            db[i] += ((va[i][0] + va[i][1]) + (va[i][2] + va[i][3])) + ((va[i][4] + va[i][5]) + (va[i][6] + va[i][7]));
            float w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float uh = (float)(signed char)(qb[i] >> (8 * j)) * sc[i];
                const float a = A.bits ? act8_relu(fmaf(ga[i], uh, be[i])) : uh;
                w[j] = mb[i] >> j & 1 ? a : 0.f;
            }
            act8_split(w, xh, xm, xl);
            d = sb + (srow + 64 * i) * AW_LD + seg;
            *reinterpret_cast<bf16x8 *>(d) = xh;
            *reinterpret_cast<bf16x8 *>(d + AW_TILE) = xm;
            *reinterpret_cast<bf16x8 *>(d + 2 * AW_TILE) = xl;
        }
    };
    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][k][e] = 0.f;
    if (s0 < s1) {
        fetch(s0);
        park();
    }
    for (long s = s0; s < s1; ++s) {
        __syncthreads();
        const bool more = s + 1 < s1;
        if (more) fetch(s + 1);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            bf16x8 a[2][3], bq[2][3];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int q = 0; q < 3; ++q) {
                    a[i][q] = *reinterpret_cast<const bf16x8 *>(sa + q * AW_TILE + (64 * wr + 32 * i + r) * AW_LD + 8 * h + 16 * ks);
                    bq[i][q] = *reinterpret_cast<const bf16x8 *>(sb + q * AW_TILE + (64 * wc + 32 * i + r) * AW_LD + 8 * h + 16 * ks);
                }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) acc[i][k] = act8_mma6(acc[i][k], a[i][0], a[i][1], a[i][2], bq[k][0], bq[k][1], bq[k][2]);
        }
        if (more) {
            __syncthreads();
            park();
        }
    }
    float *part = A.part + (long)blockIdx.y * A.N * A.K;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int col = k0 + 64 * wc + 32 * k + r;
            if (col >= A.K) continue;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int row = n0 + 64 * wr + 32 * i + 8 * (e >> 2) + 4 * h + (e & 3);
                if (row < A.N) part[(long)row * A.K + col] = acc[i][k][e];
            }
        }
    if (k0 == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float v = db[i];
            v += __shfl_xor(v, 1);
            v += __shfl_xor(v, 2);
            const int n = n0 + srow + 64 * i;
            if ((t & 3) == 0 && n < A.N) A.dbpart[(long)blockIdx.y * A.N + n] = v;
        }
    }
}

// out[i] = sum over slices, in order
__global__ __launch_bounds__(256) void p2n_act8_join_kernel(const float *__restrict__ part, long n, int slices, float *__restrict__ out) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float s = 0.f;
    for (int k = 0; k < slices; ++k) s += part[k * n + i];
    out[i] = s;
}

// ---------------------------------------------------------------- norm + ReLU alone (the end of a chain)
__global__ __launch_bounds__(256) void p2n_act8_apply_kernel(const float *__restrict__ x, long rows, int C, int Cpad, long L, const float *__restrict__ tab, float *__restrict__ out) {
    const long LB = (L + 1023) / 1024;
    const long row = blockIdx.x / LB, l0 = (blockIdx.x % LB) * 1024;
    const int c = (int)(row % C);
    const float mu = tab[c], s = tab[Cpad + c], t = tab[2 * Cpad + c];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const long l = l0 + 256 * j + threadIdx.x;
        if (l < L) {
            out[row * L + l] = act8_relu(fmaf(x[row * L + l] - mu, s, t));
        }
    }
}

// dy = [y > 0] * g and its sums; one workgroup per (channel, slice of the (cloud, group) list)
__global__ __launch_bounds__(256) void p2n_act8_dy_kernel(const float *__restrict__ g, int B, int C, long L, long NB, long per, const signed char *__restrict__ codes,
                                                          const float *__restrict__ scale, const unsigned *__restrict__ bits, float *__restrict__ dy,
                                                          float *__restrict__ part) {
    __shared__ float sh[8];
    const int c = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long n = (long)B * NB, i0 = (long)blockIdx.y * per, i1 = i0 + per < n ? i0 + per : n;
    float u = 0.f, v = 0.f;
    for (long i = i0 + wave; i < i1; i += 4) {
        const long b = i / NB, nb = i % NB, row = b * C + c, grp = row * NB + nb;
        const float s = scale[grp];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const long l = nb * ACT8_GROUP + 64 * j + lane;
            if (l >= L) continue;
            const unsigned w = bits[grp * 4 + 2 * j + (lane >> 5)];
            const float d = w >> (lane & 31) & 1 ? g[row * L + l] : 0.f;
            dy[row * L + l] = d;
            u += d;
            if (d != 0.f) v += d * ((float)codes[grp * ACT8_GROUP + 64 * j + lane] * s);
        }
    }
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        u += __shfl_xor(u, m);
        v += __shfl_xor(v, m);
    }
    if (lane == 0) { sh[wave] = u; sh[4 + wave] = v; }
    __syncthreads();
    if (threadIdx.x == 0) {
        part[((long)c * 2) * gridDim.y + blockIdx.y] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
        part[((long)c * 2 + 1) * gridDim.y + blockIdx.y] = (sh[4] + sh[5]) + (sh[6] + sh[7]);
    }
}

// ---------------------------------------------------------------- host
namespace {
struct Act8 {
    int B, K, N;             // clouds, input channels, output channels
    long L, NB;
    int Kpad, KSf, CTf, KSb, CTb;     // forward product (rows N, inner K), data gradient (rows K, inner N): k-steps, padded channel tiles
    int S;                   // slices of the statistics
    long per;
    int slices;              // of the weight gradient
    long steps, wper;
};

int act8_tiles(int rows) { return rows <= 32 ? 1 : rows <= 64 ? 2 : rows <= 128 ? 4 : 8; }   // channel tiles of a workgroup
int act8_ksteps(int k, int ct) {
    const int cks = ct >= 4 ? 1 : 4 / ct, ks = (k + 15) / 16;
    return (ks + cks - 1) / cks * cks;
}
int act8_padded(int rows, int ct) { return ((rows + 31) / 32 + ct - 1) / ct * ct; }

int act8_init(Act8 &a, const char *fn, int B, int K, long L, int N) {
    P2N_REQUIRE(B >= 1 && L >= 1 && L <= (1L << 24), "%s: bad shape B=%d L=%ld (1 to 2^24 columns a cloud)", fn, B, L);
    P2N_REQUIRE(K >= 1 && K <= ACT8_MAX_C && N >= 0 && N <= ACT8_MAX_C, "%s: %d or %d channels, not in [1,%d]", fn, K, N, ACT8_MAX_C);
    a.B = B; a.K = K; a.N = N; a.L = L; a.NB = (L + ACT8_GROUP - 1) / ACT8_GROUP;
    P2N_REQUIRE((long)B * a.NB * K < (1L << 31) && (long)B * ((L + 1023) / 1024) * K < (1L << 31), "%s: too many points", fn);
    a.Kpad = (K + 63) / 64 * 64;
    const int cf = act8_tiles(N ? N : 1), cb = act8_tiles(K);
    a.KSf = act8_ksteps(K, cf); a.CTf = act8_padded(N ? N : 1, cf);
    a.KSb = act8_ksteps(N ? N : 1, cb); a.CTb = act8_padded(K, cb);
    const long blocks = (long)B * ((L + 1023) / 1024);
    long s = 2048 / K > 1 ? 2048 / K : 1;
    if (s > blocks) s = blocks;
    if (s > 1024) s = 1024;
    a.per = (blocks + s - 1) / s;
    a.S = (int)((blocks + a.per - 1) / a.per);
    a.steps = (long)B * a.NB * 4;
    const long tiles = (long)((N + 127) / 128) * ((K + 127) / 128);
    long sl = tiles ? 512 / tiles : 1;
    if (sl < 1) sl = 1;
    if (sl > (a.steps + 15) / 16) sl = (a.steps + 15) / 16;
    a.wper = (a.steps + sl - 1) / sl;
    a.slices = (int)((a.steps + a.wper - 1) / a.wper);
    return P2N_OK;
}

struct Carve {
    char *base;
    size_t off;
    template <typename T>
    T *take(size_t n) {
        T *p = base ? (T *)(base + off) : nullptr;
        off += (n * sizeof(T) + 255) & ~(size_t)255;
        return p;
    }
};

struct FwdSpace {
    double *part;
    float *tab;
    __bf16 *img;
    size_t total;
};
FwdSpace fwd_space(const Act8 &a, char *base) {
    Carve c{base, 0};
    FwdSpace f;
    f.part = c.take<double>((size_t)2 * a.K * a.S);
    f.tab = c.take<float>((size_t)3 * a.Kpad);
    f.img = c.take<__bf16>((size_t)a.CTf * a.KSf * 1536);
    f.total = c.off;
    return f;
}

struct BwdSpace {
    float *part, *tab, *wpart, *dbpart;
    __bf16 *img;
    long nparts;
    size_t total;
};
BwdSpace bwd_space(const Act8 &a, char *base) {
    Carve c{base, 0};
    BwdSpace f;
    f.nparts = a.N ? (long)a.B * a.NB : a.S;
    f.part = c.take<float>((size_t)2 * a.K * f.nparts);
    f.tab = c.take<float>((size_t)3 * a.K);
    f.img = c.take<__bf16>((size_t)a.CTb * a.KSb * 1536);
    f.wpart = c.take<float>((size_t)a.slices * a.N * a.K);
    f.dbpart = c.take<float>((size_t)a.slices * a.N);
    f.total = c.off;
    return f;
}

int act8_split_weights(const float *W, int rows, int cols, int trans, int CTP, int KS, __bf16 *img, hipStream_t s) {
    const long n = (long)CTP * KS * 64;
    hipLaunchKernelGGL(p2n_act8_split_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, W, rows, cols, trans, CTP, KS, img);
    P2N_CHECK_HIP(hipGetLastError());
    return P2N_OK;
}

template <int IN, int EPI>
int act8_launch_gemm(const Act8Gemm &g, long groups, hipStream_t s) {
    const int ct = act8_tiles(g.rows);
    const dim3 grid((unsigned)groups, (unsigned)(g.CTP / ct)), blk(256);
    switch (ct) {
        case 1: hipLaunchKernelGGL((p2n_act8_gemm_kernel<IN, EPI, 1>), grid, blk, 0, s, g); break;
        case 2: hipLaunchKernelGGL((p2n_act8_gemm_kernel<IN, EPI, 2>), grid, blk, 0, s, g); break;
        case 4: hipLaunchKernelGGL((p2n_act8_gemm_kernel<IN, EPI, 4>), grid, blk, 0, s, g); break;
        default: hipLaunchKernelGGL((p2n_act8_gemm_kernel<IN, EPI, 8>), grid, blk, 0, s, g);
    }
    P2N_CHECK_HIP(hipGetLastError());
    return P2N_OK;
}

int act8_space_check(const char *fn, const void *p, size_t have, size_t need, const char *what) {
    if (!p || have < need) {
        p2n_set_error("%s: %s %zu bytes < required %zu", fn, what, have, need);
        return P2N_EWORKSPACE;
    }
    P2N_REQUIRE(((uintptr_t)p & 255) == 0, "%s: the %s must be 256-byte aligned", fn, what);
    return P2N_OK;
}

// statistics, tables and codes of x; returns with f.tab set (norm)
int act8_keep(const Act8 &a, const char *fn, const float *x, const float *gamma, const float *beta, float *rmean, float *rvar, float momentum,
              float eps, char *kept, const FwdSpace &f, hipStream_t s) {
    const Act8Kept k = act8_kept(a.B, a.K, a.L, gamma != nullptr);
    float *stat = (float *)(kept + k.stat);
    const long groups = (long)a.B * a.K * a.NB;
    const dim3 pgrid((unsigned)((groups + 3) / 4)), blk(256);
    if (gamma) {
        const bool frozen = momentum < 0.f;
        const double P = (double)a.B * a.L;
        if (!frozen) {
            const long blocks = (long)a.B * ((a.L + 1023) / 1024);
            hipLaunchKernelGGL(p2n_act8_stats_kernel, dim3(a.K, a.S), blk, 0, s, x, a.B, a.K, a.L, blocks, a.per, f.part);
            P2N_CHECK_HIP(hipGetLastError());
        }
        hipLaunchKernelGGL(p2n_act8_norm_kernel, dim3(a.Kpad / 64), dim3(64), 0, s, f.part, a.S, x, a.K, a.Kpad, a.L, P, gamma, beta, rmean, rvar,
                           (double)momentum, (double)eps, frozen ? 1 : 0, stat, f.tab);
        P2N_CHECK_HIP(hipGetLastError());
        hipLaunchKernelGGL(p2n_act8_pack_kernel<true>, pgrid, blk, 0, s, x, groups, a.K, a.L, a.NB, stat, gamma, beta, (signed char *)kept,
                           (float *)(kept + k.scale), (unsigned *)(kept + k.bits));
    } else {
        hipLaunchKernelGGL(p2n_act8_pack_kernel<false>, pgrid, blk, 0, s, x, groups, a.K, a.L, a.NB, nullptr, nullptr, nullptr, (signed char *)kept,
                           (float *)(kept + k.scale), nullptr);
    }
    P2N_CHECK_HIP(hipGetLastError());
    return P2N_OK;
}

int act8_norm_check(const char *fn, const Act8 &a, const float *gamma, const float *beta, const float *rmean, const float *rvar, float momentum, float eps) {
    if (!gamma) return P2N_OK;
    P2N_REQUIRE(beta && (!rmean == !rvar), "%s: a norm needs gamma and beta, and both running statistics or none", fn);
    P2N_REQUIRE(momentum <= 1.f && eps >= 0.f, "%s: momentum %g not in [0,1] (negative: running statistics) or eps %g < 0", fn, momentum, eps);
    if (momentum < 0.f) P2N_REQUIRE(rmean, "%s: frozen statistics need the running mean and variance", fn);
    else P2N_REQUIRE((double)a.B * a.L >= 2, "%s: batch statistics need more than one value per channel", fn);
    return P2N_OK;
}
}  // namespace

extern "C" size_t p2n_act8_kept_bytes(int B, int C, long L, int norm) {
    Act8 a;
    if (act8_init(a, "p2n_act8_kept_bytes", B, C, L, 0)) return 0;
    return act8_kept(B, C, L, norm).total;
}

extern "C" size_t p2n_act8_workspace_bytes(int B, int K, long L, int N) {
    Act8 a;
    if (act8_init(a, "p2n_act8_workspace_bytes", B, K, L, N)) return 0;
    const size_t f = fwd_space(a, nullptr).total, b = bwd_space(a, nullptr).total;
    return f > b ? f : b;
}

extern "C" int p2n_act8_forward(const float *x, int B, int K, long L, const float *W, const float *bias, int N, const float *gamma, const float *beta,
                                float *running_mean, float *running_var, float momentum, float eps, float *h, void *kept, size_t kept_bytes,
                                void *workspace, size_t workspace_bytes, void *stream_) {
    const char *fn = "p2n_act8_forward";
    Act8 a;
    P2N_REQUIRE(N >= 1, "%s: %d output channels", fn, N);
    TRY(act8_init(a, fn, B, K, L, N));
    P2N_REQUIRE(x && W && h, "%s: null pointer", fn);
    TRY(act8_norm_check(fn, a, gamma, beta, running_mean, running_var, momentum, eps));
    TRY(act8_space_check(fn, kept, kept_bytes, act8_kept(B, K, L, gamma != nullptr).total, "kept buffer"));
    TRY(act8_space_check(fn, workspace, workspace_bytes, fwd_space(a, nullptr).total, "workspace"));
    const FwdSpace f = fwd_space(a, (char *)workspace);
    hipStream_t s = (hipStream_t)stream_;
    const int ps = p2n_prof_begin(P2N_K_ACT8_FWD, s);
    TRY(act8_keep(a, fn, x, gamma, beta, running_mean, running_var, momentum, eps, (char *)kept, f, s));
    TRY(act8_split_weights(W, N, K, 0, a.CTf, a.KSf, f.img, s));
    Act8Gemm g = {};
    g.x = x; g.img = f.img; g.tab = f.tab; g.bias = bias; g.out = h; g.L = L; g.NB = a.NB;
    g.K = K; g.Kpad = a.Kpad; g.KS = a.KSf; g.CTP = a.CTf; g.rows = N;
    const long groups = (long)B * a.NB;
    if (gamma) TRY((act8_launch_gemm<ACT8_NORM, ACT8_OUT>(g, groups, s)));
    else TRY((act8_launch_gemm<ACT8_PLAIN, ACT8_OUT>(g, groups, s)));
    p2n_prof_end(ps, s);
    return P2N_OK;
}

extern "C" int p2n_act8_backward(const float *g, int B, int K, long L, const float *W, int N, const float *gamma, const float *beta, int frozen,
                                 const void *kept_, size_t kept_bytes, float *dx, float *dW, float *db, float *dgamma, float *dbeta, void *workspace,
                                 size_t workspace_bytes, void *stream_) {
    const char *fn = "p2n_act8_backward";
    Act8 a;
    P2N_REQUIRE(N >= 1, "%s: %d output channels", fn, N);
    TRY(act8_init(a, fn, B, K, L, N));
    P2N_REQUIRE(g && W && (!gamma || beta), "%s: null pointer", fn);
    P2N_REQUIRE(!gamma || dx || !(dgamma || dbeta), "%s: the norm's gradients need dx, through which they are formed", fn);
    const Act8Kept k = act8_kept(B, K, L, gamma != nullptr);
    TRY(act8_space_check(fn, kept_, kept_bytes, k.total, "kept buffer"));
    TRY(act8_space_check(fn, workspace, workspace_bytes, bwd_space(a, nullptr).total, "workspace"));
    const BwdSpace f = bwd_space(a, (char *)workspace);
    const char *kept = (const char *)kept_;
    const signed char *codes = (const signed char *)kept;
    const float *scale = (const float *)(kept + k.scale), *stat = (const float *)(kept + k.stat);
    const unsigned *bits = gamma ? (const unsigned *)(kept + k.bits) : nullptr;
    hipStream_t s = (hipStream_t)stream_;
    const int ps = p2n_prof_begin(P2N_K_ACT8_BWD, s);
    const long groups = (long)B * a.NB;
    if (dW || db) {
        Act8Wgrad w = {};
        w.g = g; w.codes = codes; w.scale = scale; w.bits = bits; w.gamma = gamma; w.beta = beta; w.part = f.wpart; w.dbpart = f.dbpart;
        w.L = L; w.NB = a.NB; w.steps = a.steps; w.per = a.wper; w.N = N; w.K = K;
        hipLaunchKernelGGL(p2n_act8_wgrad_kernel, dim3(((N + 127) / 128) * ((K + 127) / 128), a.slices), dim3(256), 0, s, w);
        P2N_CHECK_HIP(hipGetLastError());
        const long n = (long)N * K;
        if (dW) hipLaunchKernelGGL(p2n_act8_join_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, f.wpart, n, a.slices, dW);
        if (db) hipLaunchKernelGGL(p2n_act8_join_kernel, dim3((unsigned)((N + 255) / 256)), dim3(256), 0, s, f.dbpart, (long)N, a.slices, db);
        P2N_CHECK_HIP(hipGetLastError());
    }
    if (dx) {
        TRY(act8_split_weights(W, K, N, 1, a.CTb, a.KSb, f.img, s));
        Act8Gemm q = {};
        q.x = g; q.img = f.img; q.out = dx; q.codes = codes; q.scale = scale; q.bits = bits; q.part = f.part; q.L = L; q.NB = a.NB;
        q.K = N; q.Kpad = (N + 63) / 64 * 64; q.KS = a.KSb; q.CTP = a.CTb; q.rows = K;
        if (gamma) {
            TRY((act8_launch_gemm<ACT8_PLAIN, ACT8_DY>(q, groups, s)));
            hipLaunchKernelGGL(p2n_act8_sums_kernel, dim3(K), dim3(256), 0, s, f.part, f.nparts, K, (double)B * L, gamma, stat, frozen ? 1 : 0, dgamma, dbeta, f.tab);
            P2N_CHECK_HIP(hipGetLastError());
            hipLaunchKernelGGL(p2n_act8_dx_kernel, dim3((unsigned)((groups * K + 3) / 4)), dim3(256), 0, s, dx, groups * K, K, L, a.NB, f.tab, codes, scale);
            P2N_CHECK_HIP(hipGetLastError());
        } else {
            TRY((act8_launch_gemm<ACT8_PLAIN, ACT8_OUT>(q, groups, s)));
        }
    }
    p2n_prof_end(ps, s);
    return P2N_OK;
}

extern "C" int p2n_act8_norm_relu_forward(const float *x, int B, int C, long L, const float *gamma, const float *beta, float *running_mean,
                                          float *running_var, float momentum, float eps, float *out, void *kept, size_t kept_bytes, void *workspace,
                                          size_t workspace_bytes, void *stream_) {
    const char *fn = "p2n_act8_norm_relu_forward";
    Act8 a;
    TRY(act8_init(a, fn, B, C, L, 0));
    P2N_REQUIRE(x && out && gamma && beta, "%s: null pointer", fn);
    TRY(act8_norm_check(fn, a, gamma, beta, running_mean, running_var, momentum, eps));
    TRY(act8_space_check(fn, kept, kept_bytes, act8_kept(B, C, L, 1).total, "kept buffer"));
    TRY(act8_space_check(fn, workspace, workspace_bytes, fwd_space(a, nullptr).total, "workspace"));
    const FwdSpace f = fwd_space(a, (char *)workspace);
    hipStream_t s = (hipStream_t)stream_;
    const int ps = p2n_prof_begin(P2N_K_ACT8_FWD, s);
    TRY(act8_keep(a, fn, x, gamma, beta, running_mean, running_var, momentum, eps, (char *)kept, f, s));
    const long rows = (long)B * C;
    hipLaunchKernelGGL(p2n_act8_apply_kernel, dim3((unsigned)(rows * ((L + 1023) / 1024))), dim3(256), 0, s, x, rows, C, a.Kpad, L, f.tab, out);
    P2N_CHECK_HIP(hipGetLastError());
    p2n_prof_end(ps, s);
    return P2N_OK;
}

extern "C" int p2n_act8_norm_relu_backward(const float *g, int B, int C, long L, const float *gamma, int frozen, const void *kept_, size_t kept_bytes,
                                           float *dx, float *dgamma, float *dbeta, void *workspace, size_t workspace_bytes, void *stream_) {
    const char *fn = "p2n_act8_norm_relu_backward";
    Act8 a;
    TRY(act8_init(a, fn, B, C, L, 0));
    P2N_REQUIRE(g && gamma && dx, "%s: null pointer", fn);
    const Act8Kept k = act8_kept(B, C, L, 1);
    TRY(act8_space_check(fn, kept_, kept_bytes, k.total, "kept buffer"));
    TRY(act8_space_check(fn, workspace, workspace_bytes, bwd_space(a, nullptr).total, "workspace"));
    const BwdSpace f = bwd_space(a, (char *)workspace);
    const char *kept = (const char *)kept_;
    const signed char *codes = (const signed char *)kept;
    const float *scale = (const float *)(kept + k.scale), *stat = (const float *)(kept + k.stat);
    hipStream_t s = (hipStream_t)stream_;
    const int ps = p2n_prof_begin(P2N_K_ACT8_BWD, s);
    const long n = (long)B * a.NB, per = (n + a.S - 1) / a.S, groups = n * C;
    hipLaunchKernelGGL(p2n_act8_dy_kernel, dim3(C, a.S), dim3(256), 0, s, g, B, C, L, a.NB, per, codes, scale, (const unsigned *)(kept + k.bits), dx, f.part);
    P2N_CHECK_HIP(hipGetLastError());
    hipLaunchKernelGGL(p2n_act8_sums_kernel, dim3(C), dim3(256), 0, s, f.part, f.nparts, C, (double)B * L, gamma, stat, frozen ? 1 : 0, dgamma, dbeta, f.tab);
    P2N_CHECK_HIP(hipGetLastError());
    hipLaunchKernelGGL(p2n_act8_dx_kernel, dim3((unsigned)((groups + 3) / 4)), dim3(256), 0, s, dx, groups, C, L, a.NB, f.tab, codes, scale);
    P2N_CHECK_HIP(hipGetLastError());
    p2n_prof_end(ps, s);
    return P2N_OK;
}
