// Training layers that keep their input for the backward pass in 8 bits (gfx950).
//     h = W . a + b,   a = relu(norm(x))  or  a = x          x (B, K, L), W (N, K), h (B, N, L)
// norm is BatchNorm over the B*L points of a channel (reference point2net.py:9-34 in train() mode): mean and biased variance
// from sums in 64 bits, mu and r = 1/sqrt(var + eps) kept as float32, u = fl(fl(x - mu) * r), y = gamma*u + beta.
// Kept instead of x: the codes of u (of x without a norm) by the 8-bit rule of p2n_q8.h, one scale for 128 consecutive points of a
// (cloud, channel) row, and one bit [y > 0] for each value, so the ReLU's decisions stay exact: 1.16 bytes a value for 4.  (The
// forward product forms y from x - mu and gamma*r in one fma: within a rounding of zero it may pass a value that size whose bit is clear.)
// A NaN counts as above zero, so it goes on into everything that its value enters, on the way back too.
// The backward pass works from uh = s*q and ah = [y > 0] * max(gamma*uh + beta, 0):
//     dW = g . ah^T   db = sum g   da = W^T . g   dy = [y > 0] * da   dbeta = sum dy   dgamma = sum dy*uh
//     dx = gamma*r*(dy - dbeta/P - uh*dgamma/P),  P = B*L   (frozen statistics: gamma*r*dy;  without a norm: da)
// The reference keeps float32 activations (train.py:124-131 under autograd); the formulas above are the specification.
//
// Products of float32 operands run on the bf16 matrix cores: each operand is the exact sum of three bf16 parts (24 bits),
// and of the nine part products the six that reach 2^-16 of the largest are added in float32 -- float32 accuracy at
// 1/6 of the bf16 rate, against 1/16 for the float32 instruction.
#include <type_traits>
#include "p2n_q8.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
#define MFMAB(a, b, c) __builtin_amdgcn_mfma_f32_32x32x16_bf16((a), (b), (c), 0, 0, 0)
#define ACT8_MAX_C 1024
#define ACT8_GROUP 128
// What the next kernels do not read (codes; g at its last reading; h where it is larger than the last cache, so that none of it would be
// there for the next layer) goes past the caches, and x, g and dy stay there for the kernel that reads them next: 32 -> 64
// over 1,048,576 points: forward 79 -> 64 us, codes 44 -> 41, both gradients 119 -> 103.  A chain of layers whose h fits loses
// 1 to 2.5 % if h goes past it (256-256-256-256 over 131,072 points, h 134 MB: 1466 us a step against 1484).
#define ACT8_ONCE 2        // the buffer instructions' bit for it
#define ACT8_LAST_CACHE (256L << 20)

#define TRY(expr)                  \
    do {                           \
        const int rc_ = (expr);    \
        if (rc_) return rc_;       \
    } while (0)

// ---------------------------------------------------------------- what is kept
// For each (cloud, block of 128 points) in turn, C4 = channels rounded up to 4, NB = ceil(L / 128):
//   codes  [C][128]      a byte a value; zero behind the last point
//   scales [C4]          float32
//   bits   [4][C4]       (norm) word w: points 32w .. 32w+31, point p at bit (p >> 1) + 16 (p & 1); zero behind the last point
// each part for all blocks before the next, and mu[C], r[C] at the end.
struct Act8Kept {
    long NB;
    size_t scale, bits, stat, total;
};

static Act8Kept act8_kept(int B, int C, long L, int norm) {
    Act8Kept k;
    k.NB = (L + ACT8_GROUP - 1) / ACT8_GROUP;
    const size_t blocks = (size_t)B * k.NB, C4 = (C + 3) / 4 * 4;
    k.scale = (blocks * C * ACT8_GROUP + 255) & ~(size_t)255;
    k.bits = k.scale + ((blocks * C4 * 4 + 255) & ~(size_t)255);
    k.stat = k.bits + (norm ? (blocks * C4 * 16 + 255) & ~(size_t)255 : 0);
    k.total = k.stat + (norm ? ((size_t)C * 8 + 255) & ~(size_t)255 : 0);
    return k;
}

// loads of 2 or 4 values from any 4-byte address
typedef float f32x2u __attribute__((ext_vector_type(2), aligned(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float act8_relu(float y) { return y <= 0.f ? 0.f : y; }   // a NaN stays

// ---------------------------------------------------------------- BatchNorm statistics
// mu, r kept as float32; tab = {mu, gamma*r, beta} for the forward loader, zero behind the last channel; running statistics (unbiased
// variance) and the count of batches brought up to date.  By one lane, of the channel's sums, or (frozen) from the running statistics.
struct Act8Norm {
    const float *x, *gamma, *beta;
    float *rmean, *rvar;
    long *batches;
    double momentum, eps, P;
    int frozen, C, Cpad;
    long L;
    float *stat, *tab;
};
__device__ __forceinline__ void act8_norm_finish(const Act8Norm &A, int c, double u, double v) {
    double mean, var;
    if (A.frozen) {
        mean = A.rmean[c];
        var = A.rvar[c];
    } else {
        const double d = u / A.P;
        mean = (double)A.x[(long)c * A.L] + d;
        var = v / A.P - d * d;
        if (var < 0.0) var = 0.0;
        if (A.batches && c == 0) *A.batches += 1;
        if (A.rmean) {
            A.rmean[c] = (float)((1.0 - A.momentum) * A.rmean[c] + A.momentum * mean);
            A.rvar[c] = (float)((1.0 - A.momentum) * A.rvar[c] + A.momentum * var * (A.P / (A.P - 1.0)));
        }
    }
    const float mu = (float)mean, r = (float)(1.0 / sqrt(var + A.eps));
    A.stat[c] = mu;
    A.stat[A.C + c] = r;
    A.tab[c] = mu;
    A.tab[A.Cpad + c] = A.gamma[c] * r;
    A.tab[2 * A.Cpad + c] = A.beta[c];
}

// grid (C, S): sums of (x - pivot) and its square over a slice of the (cloud, block) list, in 64 bits, pivot = x[0][c][0].
// One reading of x: 16 x 256 x 8192 values 28 us, 4.8 TB/s.  ALONE (S = 1): the workgroup has all of its channel and finishes it
// (grid (Cpad, 1)).
template <bool ALONE>
__global__ __launch_bounds__(256) void p2n_act8_stats_kernel(const float *__restrict__ x, int B, int C, long L, long blocks, long per, double *__restrict__ part,
                                                             Act8Norm A) {
    __shared__ double sh[8];
    const int c = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long NB = (L + 2047) / 2048;                      // a block: 2048 columns of a cloud
    if (ALONE && c >= C) {
        if (threadIdx.x < 3) A.tab[threadIdx.x * A.Cpad + c] = 0.f;
        return;
    }
    const float pivot = x[(long)c * L];
    double u = 0.0, v = 0.0;
    auto add = [&](float e) __attribute__((always_inline)) {
        const double d = (double)e - (double)pivot;
        u += d;
        v += d * d;
    };
    const long b0 = (long)blockIdx.y * per, b1 = b0 + per < blocks ? b0 + per : blocks;
    for (long i = b0; i < b1; ++i) {
        const long b = i / NB, l0 = (i % NB) * 2048;
        const float *row = x + (b * C + c) * L;
        if (l0 + 2048 <= L) {
            f32x4u e[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) e[j] = *reinterpret_cast<const f32x4u *>(row + l0 + 1024 * j + 4 * threadIdx.x);
#pragma unroll
            for (int j = 0; j < 8; ++j) add(e[j >> 2][j & 3]);
        } else {
            for (long l = l0 + threadIdx.x; l < L; l += 256) add(row[l]);
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
        u = (sh[0] + sh[1]) + (sh[2] + sh[3]);
        v = (sh[4] + sh[5]) + (sh[6] + sh[7]);
        if (ALONE) {
            act8_norm_finish(A, c, u, v);
        } else {
            part[((long)c * gridDim.y + blockIdx.y) * 2] = u;
            part[((long)c * gridDim.y + blockIdx.y) * 2 + 1] = v;
        }
    }
}

// the slices' sums of a channel, by one wave
__global__ void p2n_act8_norm_kernel(const double *__restrict__ part, int S, Act8Norm A) {
    const int c = blockIdx.x, lane = threadIdx.x;
    if (c >= A.C) {
        if (lane < 3) A.tab[lane * A.Cpad + c] = 0.f;
        return;
    }
    double u = 0.0, v = 0.0;
    if (!A.frozen)
        for (int s = lane; s < S; s += 64) { u += part[((long)c * S + s) * 2]; v += part[((long)c * S + s) * 2 + 1]; }
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        u += __shfl_xor(u, m);
        v += __shfl_xor(v, m);
    }
    if (lane == 0) act8_norm_finish(A, c, u, v);
}


// ---------------------------------------------------------------- weight image of a product
// three-way split w = h + m + l: fragment (ks * CTP + ct) * 3 + part, 1 KiB: lane holds part(M[32ct + (lane&31)][16ks + 8(lane>>5) + i]),
// i < 8; M = W (rows N) or W^T (rows K); zero outside.  CTP = channel tiles rounded up to what a workgroup makes.  It is made by
// the first workgroups of a launch that the product follows anyway (a launch of its own: 4 us; by the last workgroups: 6).
struct Act8Split {
    const float *W;
    __bf16 *img;
    int rows, cols, trans, CTP, KS;
};
__device__ __forceinline__ void act8_split_rounded(const float (&v)[8], bf16x8 &h, bf16x8 &m, bf16x8 &l) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        h[j] = (__bf16)v[j];
        const float r = v[j] - (float)h[j];
        m[j] = (__bf16)r;
        l[j] = (__bf16)(r - (float)m[j]);
    }
}
__device__ __forceinline__ void act8_split_weights(const Act8Split &A, long i) {      // i: (fragment without part, lane)
    const int lane = (int)(i & 63);
    const long f = i >> 6;
    if (f >= (long)A.CTP * A.KS) return;
    const int ct = (int)(f % A.CTP), ks = (int)(f / A.CTP);
    const int row = 32 * ct + (lane & 31), k0 = 16 * ks + 8 * (lane >> 5);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int k = k0 + j;
        v[j] = row < A.rows && k < A.cols ? (A.trans ? A.W[(long)k * A.rows + row] : A.W[(long)row * A.cols + k]) : 0.f;
    }
    bf16x8 h, m, l;
    act8_split_rounded(v, h, m, l);
    bf16x8 *d = reinterpret_cast<bf16x8 *>(A.img) + f * 3 * 64 + lane;
    d[0] = h; d[64] = m; d[128] = l;
}

// ---------------------------------------------------------------- codes
// What is kept of a block of 128 points, 32 channels a workgroup and 8 a wave, a lane two neighbouring points: u, the scales, codes,
// the ReLU's bits.  The channels' maxima are formed by a halving exchange (8 registers shrink to one while lanes pair up), so lane i
// holds the maximum of channel i & 7 and one division serves eight channels.  OUT (the end of a chain): relu(y) to `out` as well.
// 16 x 256 x 8192 values: 43 us, 4.0 TB/s.  Formed by the product's workgroups instead, before their products, it costs 73: nothing
// overlaps with it there.
struct Act8Keep {
    const float *x;
    const float *stat, *gamma, *beta;    // NORM
    signed char *codes;
    float *scale;
    unsigned *bits;
    float *out;                          // OUT
    long L, NB, split_wgs;               // the first workgroups make the image
    int C, C4;
    Act8Split split;
};
template <bool NORM, bool OUT>
__global__ __launch_bounds__(256) void p2n_act8_keep_kernel(Act8Keep A) {
    const int lane = threadIdx.x & 63;
    const int c0 = blockIdx.y * 32 + 8 * __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const long blk = blockIdx.x - A.split_wgs;
    if (blk < 0) {
        if (blockIdx.y == 0) act8_split_weights(A.split, (long)blockIdx.x * 256 + threadIdx.x);
        return;
    }
    if (c0 >= A.C4) return;
    const long b = blk / A.NB, l = (blk % A.NB) * ACT8_GROUP + 2 * lane;
    const bool ok0 = l < A.L, ok1 = l + 1 < A.L;
    float v[8][2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float *row = A.x + (b * A.C + (c0 + i < A.C ? c0 + i : A.C - 1)) * A.L;
        v[i][0] = v[i][1] = 0.f;
        if (ok1) {
            const f32x2u e = *reinterpret_cast<const f32x2u *>(row + l);
            v[i][0] = e[0]; v[i][1] = e[1];
        } else if (ok0) {
            v[i][0] = row[l];
        }
    }
    unsigned word = 0;
    const int q = (lane >> 3) & 3;
    unsigned am[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = c0 + i < A.C ? c0 + i : A.C - 1;
        if (NORM) {
            const float mu = A.stat[c], r = A.stat[A.C + c], ga = A.gamma[c], be = A.beta[c];
            v[i][0] = ok0 ? (v[i][0] - mu) * r : 0.f;
            v[i][1] = ok1 ? (v[i][1] - mu) * r : 0.f;
            const float y0 = fmaf(ga, v[i][0], be), y1 = fmaf(ga, v[i][1], be);
            const unsigned long long e = __ballot(ok0 && !(y0 <= 0.f)), o = __ballot(ok1 && !(y1 <= 0.f));
            const unsigned w = ((unsigned)(e >> (16 * q)) & 0xFFFFu) | (unsigned)(o >> (16 * q)) << 16;
            word = (lane & 7) == i ? w : word;
            if (OUT && c0 + i < A.C) {
                float *row = A.out + (b * A.C + c0 + i) * A.L;
                if (ok1) *reinterpret_cast<f32x2u *>(row + l) = f32x2u{act8_relu(y0), act8_relu(y1)};
                else if (ok0) row[l] = act8_relu(y0);
            }
        }
        const unsigned a = p2n_absbits(v[i][0]), a1 = p2n_absbits(v[i][1]);
        am[i] = a > a1 ? a : a1;
    }
#pragma unroll
    for (int n = 4, m = 1; n >= 1; n >>= 1, m <<= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const bool up = lane & m;
            const unsigned keep = up ? am[2 * i + 1] : am[2 * i], give = up ? am[2 * i] : am[2 * i + 1];
            const unsigned o = (unsigned)__shfl_xor((int)give, m);
            am[i] = keep > o ? keep : o;
        }
#pragma unroll
    for (int m = 8; m < 64; m <<= 1) {
        const unsigned o = (unsigned)__shfl_xor((int)am[0], m);
        am[0] = o > am[0] ? o : am[0];
    }
    const float s = p2n_q8_scale(am[0]);                  // of channel c0 + (lane & 7)
    const P2nQ8 Q = p2n_q8_make(s);
    if (lane < 8 && c0 + lane < A.C4) A.scale[blk * A.C4 + c0 + lane] = c0 + lane < A.C ? s : 0.f;
    if (NORM && lane < 32 && c0 + (lane & 7) < A.C4) A.bits[(blk * 4 + q) * A.C4 + c0 + (lane & 7)] = c0 + (lane & 7) < A.C ? word : 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (c0 + i >= A.C) break;
        P2nQ8 R;
        R.s = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(Q.s), i));
        R.up = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(Q.up), i));
        R.inv = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(Q.inv), i));
        float e[4] = {v[i][0], v[i][1], 0.f, 0.f};
        int code[1];
        p2n_q8_pack(e, R, code);
        if (!(R.s == R.s)) code[0] = 0;
        __builtin_nontemporal_store((unsigned short)code[0], reinterpret_cast<unsigned short *>(A.codes + (blk * A.C + c0 + i) * ACT8_GROUP + 2 * lane));
    }
}

// ---------------------------------------------------------------- products over points
// D = M . X, lane = point, registers = channels.  A workgroup takes 128 points (one group of a cloud), a wave 32 of them and all of
// CT*32 output channels; the weight fragments pass through LDS (a ring of three, LDS-DMA), X through registers.  Six part products a
// multiply-add: the matrix cores are the bound with many channels (256 -> 256 over 131,072 points: 104 us forward, 990 TFLOP/s of part
// products; 122 us with the backward's epilogue), memory with few (32 -> 64 over 1,048,576: 64 to 67 us, 6 TB/s).
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
    int K, Kpad, KS, CTP, rows, rows4;
};
enum { ACT8_PLAIN = 0, ACT8_NORM = 1 };     // operand
enum { ACT8_OUT = 0, ACT8_DY = 1, ACT8_OUT_ONCE = 2 };      // epilogue

typedef __attribute__((address_space(3))) void act8_lds_t;

// bytes from base on that may be reached; none where base lies past the end (a step behind the last point of a cloud).  An offset of
// ACT8_BEHIND is past every end.
#define ACT8_BEHIND 0xFFFFFFF0L
__device__ __forceinline__ __amdgpu_buffer_rsrc_t act8_rsrc(const void *base, long bytes) {
    const long n = bytes < 0 ? 0 : bytes < ACT8_BEHIND ? bytes : ACT8_BEHIND;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, (int)n, 0x00020000);
}

// the six products of the three parts, the small ones first: l.h, h.l, m.m, m.h, h.m, h.h
__device__ constexpr int act8_first(int c) { return c == 0 ? 2 : c == 1 || c >= 4 ? 0 : 1; }
__device__ constexpr int act8_second(int c) { return c == 1 ? 2 : c == 2 || c == 4 ? 1 : 0; }

// The matrix cores cut the low bits of a sum towards minus infinity (measured: the mean of h is off by -1.5e-8 of its deviation at
// 256 channels whatever its sign, the float32 instruction's by 3e-11), and a sum over 10^5 points adds that up.  Half of the points go
// through with their sign turned round, so the cuts cancel.
__device__ __forceinline__ float act8_flip(float v, unsigned flip) { return __uint_as_float(__float_as_uint(v) ^ flip); }

// Three parts of 8 values, cut instead of rounded: a part is the upper half of a float32, what it leaves is exact, and the third holds
// the rest: bit operations and exact subtractions.  The dropped products stay under 2^-21 of the product, 2^-23 on average.
__device__ __forceinline__ void act8_split(const float (&v)[8], bf16x8 &h, bf16x8 &m, bf16x8 &l) {
    i32x4 ph, pm, pl;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned a0 = __float_as_uint(v[2 * i]), a1 = __float_as_uint(v[2 * i + 1]);
        const float r0 = v[2 * i] - __uint_as_float(a0 & 0xFFFF0000u), r1 = v[2 * i + 1] - __uint_as_float(a1 & 0xFFFF0000u);
        const unsigned b0 = __float_as_uint(r0), b1 = __float_as_uint(r1);
        const float s0 = r0 - __uint_as_float(b0 & 0xFFFF0000u), s1 = r1 - __uint_as_float(b1 & 0xFFFF0000u);
        ph[i] = (int)__builtin_amdgcn_perm(a1, a0, 0x07060302u);
        pm[i] = (int)__builtin_amdgcn_perm(b1, b0, 0x07060302u);
        pl[i] = (int)__builtin_amdgcn_perm(__float_as_uint(s1), __float_as_uint(s0), 0x07060302u);
    }
    h = __builtin_bit_cast(bf16x8, ph);
    m = __builtin_bit_cast(bf16x8, pm);
    l = __builtin_bit_cast(bf16x8, pl);
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

// k-steps of 16 in a chunk of the weights: 6 to 24 fragments
__host__ __device__ constexpr int act8_chunk(int CT) { return CT >= 4 ? 1 : 2; }

// TABK: channels that the norm's table in LDS has room for; 512 leaves room for two workgroups on a CU at 256 output channels
template <int IN, int EPI, int CT, int TABK>
__global__ __launch_bounds__(256, CT <= 4 ? 3 : TABK <= 512 ? 2 : 1) void p2n_act8_gemm_kernel(Act8Gemm A) {
    constexpr int CKS = act8_chunk(CT);
    constexpr int F = CKS * CT * 3, FW = (F + 3) / 4;      // fragments of a chunk, of a wave
    __shared__ __attribute__((aligned(16))) char wbuf[3][F * 1024];
    __shared__ __attribute__((aligned(16))) float tab[IN == ACT8_NORM ? 3 * TABK : 4];
    __shared__ float red[EPI == ACT8_DY ? 4 * 2 * 32 * CT : 1];
    __shared__ float bias[EPI != ACT8_DY ? 32 * CT : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int p = lane & 31, h = lane >> 5;
    const long b = blockIdx.x / A.NB, nb = blockIdx.x % A.NB, l = nb * ACT8_GROUP + 32 * wave + p;
    const bool valid = l < A.L;
    const int ct0 = blockIdx.y * CT;                 // first channel tile of this workgroup
    const unsigned flip = (unsigned)(p & 1) << 31;   // see act8_flip
    const int nchunk = A.KS / CKS;
    const float *xb = A.x + b * A.K * A.L;
    const unsigned off = (unsigned)((8 * h * A.L + (valid ? l : A.L - 1)) * 4);
    if (IN == ACT8_NORM)
        for (int i = threadIdx.x; i < 3 * A.Kpad; i += 256) tab[i] = A.tab[i];
    if (EPI != ACT8_DY && (int)threadIdx.x < 32 * CT)
        bias[threadIdx.x] = A.bias && 32 * ct0 + (int)threadIdx.x < A.rows ? A.bias[32 * ct0 + threadIdx.x] : 0.f;

    auto stage = [&](int c, int slot) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t rs = act8_rsrc(A.img, (long)A.CTP * A.KS * 3 * 1024);
#pragma unroll
        for (int i = 0; i < FW; ++i) {
            const int g = wave * FW + i, f = g < F ? g : F - 1;   // fragment of the chunk: k-step f / (3 CT), the rest in image order
            const int ks = c * CKS + f / (3 * CT);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (act8_lds_t *)(wbuf[slot] + f * 1024), 16, lane * 16,
                                                     ((ks * A.CTP + ct0) * 3 + f % (3 * CT)) * 1024, 0, 0);
        }
    };
    float raw[2][CKS][8];
    auto fetch = [&](int c, float (&raw)[CKS][8]) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < CKS; ++s) {
            const int k0 = 16 * (c * CKS + s);
            const long left = (long)(A.K - k0) * A.L * 4;
            const __amdgpu_buffer_rsrc_t rs = act8_rsrc(xb + (long)k0 * A.L, left);   // rows past the last read as zero
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[s][i] = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, off + (unsigned)(i * A.L * 4), 0, 0));
        }
    };
    f32x16 acc[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[ct][e] = 0.f;
    // Chunks c+1 and c+2 are on their way while chunk c is multiplied: a load from memory takes about as long as one chunk's products.
    // Every chunk issues GROUP vector-memory operations, in order, so "at most GROUP outstanding" means chunk c has arrived.
    // (The last two iterations fetch the last chunk again: the count stays the same, nobody reads it.)
    constexpr int GROUP = FW + 8 * CKS;
    static_assert(GROUP < 64, "the counter holds six bits");
    int slot = 0;
    auto body = [&](int c, float (&raw)[CKS][8]) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt((GROUP & 15) | (7 << 4) | (0 << 8) | ((GROUP >> 4) << 14));
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();                 // every wave's part of chunk c is in LDS, and nobody reads chunk c-1 any more
        asm volatile("" ::: "memory");
        bf16x8 xh[CKS], xm[CKS], xl[CKS];
#pragma unroll
        for (int s = 0; s < CKS; ++s) {
            if (IN == ACT8_NORM) {
                const int k = 16 * (c * CKS + s) + 8 * h;
#pragma unroll
                for (int i = 0; i < 8; ++i) raw[s][i] = act8_relu(fmaf(raw[s][i] - tab[k + i], tab[A.Kpad + k + i], tab[2 * A.Kpad + k + i]));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[s][i] = act8_flip(raw[s][i], flip);
            act8_split(raw[s], xh[s], xm[s], xl[s]);
        }
        const int ahead = c + 2 < nchunk ? c + 2 : nchunk - 1;
        stage(ahead, slot >= 1 ? slot - 1 : 2);       // (slot + 2) % 3
        fetch(ahead, raw);
        // two channel tiles at a time (independent sums), their fragments read one pair ahead
        __builtin_amdgcn_sched_barrier(0);
        const bf16x8 *w = reinterpret_cast<const bf16x8 *>(wbuf[slot]) + lane;
        constexpr int NT = CKS * CT, PW = NT < 2 ? 1 : 2, NP = NT / PW;
        bf16x8 f[2][PW][3];
#pragma unroll
        for (int u = 0; u < PW; ++u)
#pragma unroll
            for (int q = 0; q < 3; ++q) f[0][u][q] = w[(u * 3 + q) * 64];
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            if (i + 1 < NP) {
#pragma unroll
                for (int u = 0; u < PW; ++u)
#pragma unroll
                    for (int q = 0; q < 3; ++q) f[(i + 1) & 1][u][q] = w[(((i + 1) * PW + u) * 3 + q) * 64];
            }
#pragma unroll
            for (int q = 0; q < 6; ++q)
#pragma unroll
                for (int u = 0; u < PW; ++u) {
                    const int t = i * PW + u, ks = t / CT, ct = t % CT;
                    const bf16x8 xq = act8_second(q) == 2 ? xl[ks] : act8_second(q) == 1 ? xm[ks] : xh[ks];
                    acc[ct] = MFMAB(f[i & 1][u][act8_first(q)], xq, acc[ct]);
                }
        }
        __builtin_amdgcn_sched_group_barrier(0x100, 3 * PW * (NP > 1 ? 2 : 1), 0);      // LDS reads
#pragma unroll
        for (int i = 0; i + 2 < NP; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, 6 * PW, 0);                       // matrix products
            __builtin_amdgcn_sched_group_barrier(0x100, 3 * PW, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, 6 * PW * (NP > 1 ? 2 : 1), 0);
        __builtin_amdgcn_sched_barrier(0);
        slot = slot == 2 ? 0 : slot + 1;
    };
    __syncthreads();                                  // the table; from here on waits are counted by hand
    stage(0, 0);
    fetch(0, raw[0]);
    __builtin_amdgcn_sched_barrier(0);
    stage(nchunk > 1 ? 1 : 0, 1);
    fetch(nchunk > 1 ? 1 : 0, raw[1]);
    __builtin_amdgcn_sched_barrier(0);
    int c = 0;
#pragma unroll 1
    for (; c + 1 < nchunk; c += 2) {
        body(c, raw[0]);
        body(c + 1, raw[1]);
    }
    if (c < nchunk) body(c, raw[0]);
    __builtin_amdgcn_s_waitcnt(7 << 4);               // nothing may be on its way into LDS when the workgroup ends
    asm volatile("" ::: "memory");
    // what was kept of a channel tile, one tile ahead of its use: a lane takes 16 codes of a channel and its scale or its bits, and they turn
    // round in LDS (the weights' place, the wave's own 1280 bytes): scales, bits, codes by channel.  A lane reading its own point's bytes
    // from memory keeps the return path busy for as long as the products take.
    struct Meta {
        i32x4 q;
        unsigned k;
    } meta[2];
    auto fetch_meta = [&](Meta &M, int ct) __attribute__((always_inline)) {
        const long blk = blockIdx.x;
        const int row = 32 * (ct0 + ct) + p, c = row < A.rows ? row : A.rows - 1;
        M.q = *reinterpret_cast<const i32x4 *>(A.codes + (blk * A.rows + c) * ACT8_GROUP + 32 * wave + 16 * h);
        M.k = h ? A.bits[(blk * 4 + wave) * A.rows4 + c] : reinterpret_cast<const unsigned *>(A.scale)[blk * A.rows4 + c];
    };
    unsigned *const kept = reinterpret_cast<unsigned *>(wbuf[0]) + wave * 320;
    if (EPI == ACT8_DY) {
        fetch_meta(meta[0], 0);
        __syncthreads();                              // every wave has read its last weights
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        const int r0 = 32 * (ct0 + ct);
        if (r0 >= A.rows) continue;
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[ct][e] = act8_flip(acc[ct][e], flip);
        const __amdgpu_buffer_rsrc_t ro = act8_rsrc(A.out + (b * A.rows + r0) * A.L, (long)(A.rows - r0) * A.L * 4);
        const unsigned oo = (unsigned)((4 * h * A.L + l) * 4);
        if (EPI == ACT8_DY) {
            float s1[16], s2[16];
            const int bit = (p >> 1) + 16 * (p & 1);
            const Meta &M = meta[ct & 1];
            kept[lane] = M.k;
            *reinterpret_cast<i32x4 *>(kept + 64 + 8 * p + 4 * h) = M.q;
            if (ct + 1 < CT) fetch_meta(meta[(ct + 1) & 1], ct + 1);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const i32x4 sc = *reinterpret_cast<const i32x4 *>(kept + 8 * q + 4 * h), w = *reinterpret_cast<const i32x4 *>(kept + 32 + 8 * q + 4 * h);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int e = 4 * q + j;
                    const bool on = w[j] >> bit & 1;                             // rows past the last one are not stored
                    const float uh = (float)reinterpret_cast<const signed char *>(kept + 64 + 8 * (8 * q + 4 * h + j))[p] * __int_as_float(sc[j]);
                    const float dy = on ? acc[ct][e] : 0.f;
                    acc[ct][e] = dy;
                    s1[e] = dy;
                    s2[e] = on ? dy * uh : 0.f;
                }
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
                if (EPI != ACT8_DY) v += bias[32 * ct + 8 * (e >> 2) + 4 * h + (e & 3)];
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(v), ro, oo + (unsigned)((8 * (e >> 2) + (e & 3)) * A.L * 4), 0, EPI == ACT8_OUT_ONCE ? ACT8_ONCE : 0);
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
struct Act8Sums {
    const float *part;             // [C][2][n]
    long n;
    int C, frozen;
    double P;
    const float *gamma, *stat;
    float *dgamma, *dbeta;
    float *tab;
};
// of a channel's two sums: dbeta, dgamma, and {gamma*r, m1, m2} for dx
__device__ __forceinline__ void act8_sums_finish(const Act8Sums &A, int c, double u, double v, bool write, float (&t)[3]) {
    if (write && A.dbeta) A.dbeta[c] = (float)u;
    if (write && A.dgamma) A.dgamma[c] = (float)v;
    t[0] = A.gamma[c] * A.stat[A.C + c];
    t[1] = A.frozen ? 0.f : (float)(u / A.P);
    t[2] = A.frozen ? 0.f : (float)(v / A.P);
}
// a row's partials in 64 bits and in order
__global__ __launch_bounds__(256) void p2n_act8_sums_kernel(Act8Sums A) {
    __shared__ double sh[8];
    const int c = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double u = 0.0, v = 0.0;
    for (long i = threadIdx.x; i < A.n; i += 256) {
        u += A.part[((long)c * 2) * A.n + i];
        v += A.part[((long)c * 2 + 1) * A.n + i];
    }
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        u += __shfl_xor(u, m);
        v += __shfl_xor(v, m);
    }
    if (lane == 0) { sh[wave] = u; sh[4 + wave] = v; }
    __syncthreads();
    if (threadIdx.x == 0) {
        float t[3];
        act8_sums_finish(A, c, (sh[0] + sh[1]) + (sh[2] + sh[3]), (sh[4] + sh[5]) + (sh[6] + sh[7]), true, t);
#pragma unroll
        for (int i = 0; i < 3; ++i) A.tab[i * A.C + c] = t[i];
    }
}

// dx = gamma*r*(dy - m1 - uh*m2), in place (frozen: gamma*r*dy, where a NaN of the scale has no part): a workgroup takes 32 channels of a block of 128 points, a thread four points of four channels.
// FEW: the sums are formed here too, by every workgroup for its channels (eight threads a channel), the first of a row writes them down.
#define ACT8_FEW 64
template <bool FEW>
__global__ __launch_bounds__(256) void p2n_act8_dx_kernel(float *__restrict__ dy, int C, int C4, long L, long NB, Act8Sums A,
                                                          const signed char *__restrict__ codes, const float *__restrict__ scale) {
    __shared__ float own[FEW ? 96 : 1];
    if (FEW) {
        const int c = blockIdx.y * 32 + (threadIdx.x >> 3), cc = c < C ? c : C - 1;
        double u = 0.0, v = 0.0;
        for (int i = threadIdx.x & 7; i < (int)A.n; i += 8) {
            u += A.part[((long)cc * 2) * A.n + i];
            v += A.part[((long)cc * 2 + 1) * A.n + i];
        }
#pragma unroll
        for (int m = 4; m > 0; m >>= 1) {
            u += __shfl_xor(u, m);
            v += __shfl_xor(v, m);
        }
        float t[3];
        act8_sums_finish(A, cc, u, v, blockIdx.x == 0 && c < C && (threadIdx.x & 7) == 0, t);
        if ((threadIdx.x & 7) == 0)
#pragma unroll
            for (int i = 0; i < 3; ++i) own[32 * i + (threadIdx.x >> 3)] = t[i];
        __syncthreads();
    }
    const long blk = blockIdx.x, b = blk / NB, l0 = (blk % NB) * ACT8_GROUP;
    const int p = 4 * (threadIdx.x & 31);
    const bool whole = l0 + p + 4 <= L;
    float *d[4];
    f32x4 v[4];
    int q[4], c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c[i] = blockIdx.y * 32 + 8 * i + (threadIdx.x >> 5);
        const int cc = c[i] < C ? c[i] : C - 1;
        d[i] = dy + (b * C + cc) * L + l0 + p;
        q[i] = *reinterpret_cast<const int *>(codes + (blk * C + cc) * ACT8_GROUP + p);
        if (whole) v[i] = *reinterpret_cast<const f32x4u *>(d[i]);
        else
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i][j] = l0 + p + j < L ? d[i][j] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (c[i] >= C) continue;
        const float *t = FEW ? own + (c[i] & 31) : A.tab + c[i];
        const float a = t[0], m1 = t[FEW ? 32 : C], m2 = t[FEW ? 64 : 2 * C], s = A.frozen ? 0.f : scale[blk * C4 + c[i]];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] = a * (v[i][j] - m1 - (float)(signed char)(q[i] >> (8 * j)) * s * m2);
        if (whole) *reinterpret_cast<f32x4u *>(d[i]) = v[i];
        else
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (l0 + p + j < L) d[i][j] = v[i][j];
    }
}

// ---------------------------------------------------------------- weight gradient
// dW[n][k] = sum over points g[n] * ah[k]: lane = row of either operand, both are rows of consecutive points, and the order of the
// points inside a product is free as long as both operands agree.  A wave makes 32 RT x 32 CT of dW over its share of the
// points, 32 at a time, a lane 16 of them: its codes are one 16-byte load, its g passes through a piece of
// LDS that belongs to the wave alone (no barrier): it is read in whole cache lines, eight lanes a row (a lane reading its own row's
// bytes keeps the address unit busy for 113 cycles an instruction), and handed over as rows.  The four waves of a
// workgroup are added in LDS, the workgroups by a second kernel, both in order.
struct Act8Wgrad {
    const float *g;        // (B, N, L)
    const signed char *codes;
    const float *scale;
    const unsigned *bits;  // NULL: a = uh
    const float *gamma, *beta;
    float *part;           // [slices][N * K + N]: dW, db
    long L, NB;
    int N, K, K4, ntc, slices, steps;        // steps of 32 points in all
};

// neighbouring workgroups go to the eight dies in turn: the tiles of one slice stay on one die, whose L2 then holds its rows
struct Act8Place {
    int tile, slice;
};
__device__ __forceinline__ Act8Place act8_place(const Act8Wgrad &A) {
    const int nt = gridDim.x / A.slices, w8 = blockIdx.x >> 3, full = A.slices / 8 * 8, i = (int)blockIdx.x - full * nt;
    return i < 0 ? Act8Place{w8 % nt, w8 / nt * 8 + (int)(blockIdx.x & 7)} : Act8Place{i % nt, full + i / nt};
}

// Waves take turns: those that run at the same time read neighbouring lines of the same rows (shares of consecutive steps
// instead scatter the card's reads over as many pages of memory as there are rows in flight).
struct Act8Step {
    int b, q;                           // cloud, 32 points in it
};
struct Act8Turn {
    int b, q, spc;                      // clouds, pieces between a wave's steps; steps of a cloud
    __device__ __forceinline__ Act8Turn(const Act8Wgrad &A, int waves) : spc((int)(4 * A.NB)) {      // waves that share a tile
        b = waves / spc;
        q = waves % spc;
    }
    __device__ __forceinline__ Act8Step after(Act8Step s) const {
        s.b += b;
        s.q += q;
        if (s.q >= spc) { s.q -= spc; s.b += 1; }
        return s;
    }
};

// what was kept of a lane's channels: 16 codes each, scale, bits
template <int CT>
struct Act8Codes {
    i32x4 q[CT];
    float s[CT];
    unsigned m[CT];
};
template <int CT, bool NORM>
__device__ __forceinline__ void act8_codes(const Act8Wgrad &A, Act8Step s, int h, const int (&krow)[CT], Act8Codes<CT> &M) {
    const long blk = s.b * A.NB + (s.q >> 2);
    const int w = s.q & 3;
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        M.q[t] = *reinterpret_cast<const i32x4 *>(A.codes + (blk * A.K + krow[t]) * ACT8_GROUP + 32 * w + 16 * h);
        M.s[t] = A.scale[blk * A.K4 + krow[t]];
        M.m[t] = NORM ? A.bits[(blk * 4 + w) * A.K4 + krow[t]] : 0u;
    }
}

// eight points of a channel: their ah as an operand, its sign turned round in every other share (act8_flip; ah of a norm is not negative).
// cs = gamma * scale, mb: the lane's bits from its first point's on
template <bool NORM>
__device__ __forceinline__ void act8_operand(const i32x4 &q, int j, float cs, float be, unsigned mb, unsigned flip, bf16x8 (&w)[3]) {
    float v[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        const float c = (float)(signed char)(q[2 * j + (x >> 2)] >> (8 * (x & 3)));
        if (NORM) {
            const float y = fmaxf(fmaf(cs, c, be), 0.f);
            const unsigned on = (unsigned)((int)(mb << (31 - ((4 * j + (x >> 1)) + 16 * (x & 1)))) >> 31);
            v[x] = __uint_as_float((__float_as_uint(y) & on) | flip);
        } else {
            v[x] = act8_flip(c * cs, flip);
        }
    }
    act8_split(v, w[0], w[1], w[2]);
}

// What makes a column of dW NaN where the operand's ReLU does not let a NaN through (the maximum with zero takes it for one): a NaN of beta
// from the start, and at every step a NaN of gamma * scale.
template <bool NORM>
__device__ __forceinline__ float act8_poison(float be) { return NORM && be != be ? be : 0.f; }

// the shares of four waves, added in order: a quarter of the tile's registers at a time, all waves at once
template <int RT, int CT>
__device__ __forceinline__ void act8_wgrad_end(const Act8Wgrad &A, float *join, const f32x16 (&acc)[RT][CT], float (&db)[RT], const float (&poison)[CT],
                                               unsigned flip, int slice, int n0, int k0) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 31, h = lane >> 5;
#pragma unroll
    for (int t = 0; t < RT; ++t) db[t] += __shfl_xor(db[t], 32);
    float *part = A.part + (long)slice * (A.N * A.K + A.N);
    constexpr int Q = RT * CT * 4;          // registers of a quarter
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        __syncthreads();                    // the last rows (c = 0), the last quarter have been read
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            const int v = c * Q + i, tk = v / 16, e = v % 16;
            join[(wave * Q + i) * 64 + lane] = act8_flip(acc[tk / CT][tk % CT][e], flip) + poison[tk % CT];
        }
        if (c == 0 && h == 0)
#pragma unroll
            for (int t = 0; t < RT; ++t) join[RT * CT * 1024 + (wave * RT + t) * 32 + r] = db[t];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < Q / 4; ++i) {
            const int o = i * 256 + tid, v = c * Q + o / 64, tk = v / 16, e = v % 16, ln = o & 63;
            const int row = n0 + 32 * (tk / CT) + 8 * (e >> 2) + 4 * (ln >> 5) + (e & 3), col = k0 + 32 * (tk % CT) + (ln & 31);
            const float sum = ((join[o] + join[o + Q * 64]) + join[o + 2 * Q * 64]) + join[o + 3 * Q * 64];
            if (row < A.N && col < A.K) part[(long)row * A.K + col] = sum;
        }
        if (c == 0 && k0 == 0 && tid < 32 * RT && n0 + tid < A.N) {
            const float *d = join + RT * CT * 1024 + tid;
            part[(long)A.N * A.K + n0 + tid] = ((d[0] + d[32 * RT]) + d[64 * RT]) + d[96 * RT];
        }
    }
}
constexpr int act8_join_floats(int rt, int ct) { return rt * ct * 1024 + 4 * 32 * rt; }

// up to 64 x 64 a wave, two waves or more on a SIMD; the next step's g and codes wait in registers (for more than 64 channels on a side)
template <int RT, int CT, bool NORM>
__global__ __launch_bounds__(256, 2) void p2n_act8_wgrad_kernel(Act8Wgrad A) {
    constexpr int BUF = RT * 4096, JOIN = act8_join_floats(RT, CT) * 4;      // bytes; 32 RT rows of 32 points
    __shared__ __attribute__((aligned(16))) char lds[4 * BUF > JOIN ? 4 * BUF : JOIN];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int r = lane & 31, h = lane >> 5;
    const Act8Place at = act8_place(A);
    const int tile = at.tile, slice = at.slice;
    const int n0 = tile / A.ntc * 32 * RT, k0 = tile % A.ntc * 32 * CT;
    const int turn = A.slices * 4;
    const Act8Turn take(A, turn);
    const int first = slice * 4 + wave;
    const unsigned flip = (unsigned)((slice * 4 + wave) & 1) << 31;       // every other share with its sign turned round (act8_flip)
    const bool want_db = k0 == 0;
    int krow[CT];
    float ga[CT], be[CT], poison[CT], db[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) db[i] = 0.f;
#pragma unroll
    for (int i = 0; i < CT; ++i) {
        const int k = k0 + 32 * i + r;
        krow[i] = k < A.K ? k : A.K - 1;
        ga[i] = NORM ? A.gamma[krow[i]] : 1.f;
        be[i] = NORM ? A.beta[krow[i]] : 0.f;
        poison[i] = act8_poison<NORM>(be[i]);
    }
    f32x16 acc[RT][CT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int k = 0; k < CT; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][k][e] = 0.f;
    // LDS image of a step: row R's 16-byte piece q (points 4q .. 4q+3) lies in slot q ^ (R >> 1 & 7) of the row, so that the 16 rows of a
    // read fall into different banks.  Load i fills rows 8i .. 8i+7: lane -> row lane >> 3, piece lane & 7.
    char *const mine = lds + wave * BUF;
    const int drow = lane >> 3, slot = (lane & 7) ^ (lane >> 4);
    int qn[CT][4];
    float sn[CT];
    unsigned mn[CT];
    auto meta = [&](Act8Step s) __attribute__((always_inline)) {
        const long blk = s.b * A.NB + (s.q >> 2);
        const int w = s.q & 3;
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            const i32x4 q = *reinterpret_cast<const i32x4 *>(A.codes + (blk * A.K + krow[t]) * ACT8_GROUP + 32 * w + 16 * h);
#pragma unroll
            for (int x = 0; x < 4; ++x) qn[t][x] = q[x];
            sn[t] = A.scale[blk * A.K4 + krow[t]];
            mn[t] = NORM ? A.bits[(blk * 4 + w) * A.K4 + krow[t]] : 0u;
        }
    };
    f32x4 vn[RT * 4];
    auto rows = [&](Act8Step s) __attribute__((always_inline)) {
        const long b = s.b, l0 = (long)s.q * 32, l = l0 + 4 * (lane & 7);
        const bool tail = l0 + 32 > A.L;
#pragma unroll
        for (int i = 0; i < RT * 4; ++i) {
            const int n = n0 + 8 * i + drow;
            const float *p = A.g + (b * A.N + (n < A.N ? n : A.N - 1)) * A.L + l;      // rows past the last one read the last one
            if (!tail) vn[i] = *reinterpret_cast<const f32x4u *>(p);
            else
#pragma unroll
                for (int x = 0; x < 4; ++x) vn[i][x] = l + x < A.L ? p[x] : 0.f;
        }
    };
    Act8Step step = {first / take.spc, first % take.spc};
    if (first < A.steps) {
        rows(step);
        meta(step);
    }
#pragma unroll 1
    for (int s = first; s < A.steps; s += turn) {
#pragma unroll
        for (int i = 0; i < RT * 4; ++i) *reinterpret_cast<f32x4 *>(mine + i * 1024 + drow * 128 + (slot ^ (4 * (i & 1))) * 16) = vn[i];
        int q[CT][4];
        float cs[CT];
        unsigned mb[CT];
#pragma unroll
        for (int t = 0; t < CT; ++t) {
#pragma unroll
            for (int x = 0; x < 4; ++x) q[t][x] = qn[t][x];
            cs[t] = ga[t] * sn[t];
            poison[t] += cs[t] * 0.f;                       // NaN with a NaN scale
            mb[t] = mn[t] >> (8 * h);                       // points 16h .. 16h+15: bits 8h .. of either half-word
        }
        const Act8Step next = take.after(step);
        if (s + turn < A.steps) {
            rows(next);
            meta(next);
        }
        step = next;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            bf16x8 a[RT][3], w[CT][3];
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                float va[8];
                const char *row = mine + (32 * t + r) * 128;
                const int key = r >> 1 & 7;
                const f32x4 e0 = *reinterpret_cast<const f32x4 *>(row + ((4 * h + 2 * j) ^ key) * 16);
                const f32x4 e1 = *reinterpret_cast<const f32x4 *>(row + ((4 * h + 2 * j + 1) ^ key) * 16);
#pragma unroll
                for (int x = 0; x < 4; ++x) { va[x] = e0[x]; va[4 + x] = e1[x]; }
                if (want_db) db[t] += ((va[0] + va[1]) + (va[2] + va[3])) + ((va[4] + va[5]) + (va[6] + va[7]));
#pragma unroll
                for (int x = 0; x < 8; ++x) va[x] = act8_flip(va[x], flip);
                act8_split(va, a[t][0], a[t][1], a[t][2]);
            }
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                float v[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const float c = (float)(signed char)(q[t][2 * j + (x >> 2)] >> (8 * (x & 3)));
                    if (NORM) {
                        const float y = fmaxf(fmaf(cs[t], c, be[t]), 0.f);
                        const int on = (int)(mb[t] << (31 - ((4 * j + (x >> 1)) + 16 * (x & 1)))) >> 31;
                        v[x] = __int_as_float(__float_as_int(y) & on);
                    } else {
                        v[x] = c * cs[t];
                    }
                }
                act8_split(v, w[t][0], w[t][1], w[t][2]);
            }
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int k = 0; k < CT; ++k)
#pragma unroll
                    for (int c = 0; c < 6; ++c) acc[t][k] = MFMAB(a[t][act8_first(c)], w[k][act8_second(c)], acc[t][k]);
        }
    }
    act8_wgrad_end<RT, CT>(A, reinterpret_cast<float *>(lds), acc, db, poison, flip, slice, n0, k0);
}

// 128 x 128 a wave, the only one on its SIMD: splitting the operands (8 to 9 vector instructions a product) has to go on while the matrix
// core works, so the operands of the next 24 products are formed between the products of the present 24, and a quarter of the other
// side's next ones with them (256 x 256 over 131,072 points with the join, in a stream of calls: 117 us; 127 on the card where forming
// each 16 points' operands first took 141; alone in a kernel trace 142 + 9).
// g comes by LDS-DMA, a step ahead, codes into registers, two ahead.  Rows of g start on 16 bytes, L a multiple of 4.
template <bool NORM>
__global__ __launch_bounds__(256, 1) void p2n_act8_wgrad_wide_kernel(Act8Wgrad A) {
    constexpr int BUF = 4096;                                                // floats: 128 rows of 32 points
    __shared__ __attribute__((aligned(16))) float lds[8 * BUF];
    static_assert(8 * BUF >= act8_join_floats(4, 4), "the shares pass through the same memory");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int r = lane & 31, h = lane >> 5;
    const Act8Place at = act8_place(A);
    const int n0 = at.tile / A.ntc * 128, k0 = at.tile % A.ntc * 128;
    const int first = at.slice * 4 + wave, stride = A.slices * 4;
    const Act8Turn turn(A, stride);
    const unsigned flip = (unsigned)(first & 1) << 31;
    int krow[4];
    float ga[4], be[4], poison[4], db[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = k0 + 32 * i + r;
        krow[i] = k < A.K ? k : A.K - 1;
        ga[i] = NORM ? A.gamma[krow[i]] : 1.f;
        be[i] = NORM ? A.beta[krow[i]] : 0.f;
        poison[i] = act8_poison<NORM>(be[i]);
        db[i] = 0.f;
    }
    f32x16 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][k][e] = 0.f;
    // a step's rows in LDS as above; instruction i fills rows 8i .. 8i+7, lane -> row lane >> 3, slot lane & 7.  The resource ends with the
    // cloud: rows past the last one read as zero, and so do pieces behind a row's last point, which are given an offset past any end.
    float *const mine = lds + wave * 2 * BUF;
    const int piece = (lane & 7) ^ (lane >> 4);
    const unsigned drow = (unsigned)((lane >> 3) * A.L * 4);
    const long eight = 8 * A.L;
    auto dma = [&](Act8Step s, int buf) __attribute__((always_inline)) {
        const long l0 = (long)s.q * 32;
        const float *src = A.g + ((long)s.b * A.N + n0) * A.L + l0;
        long size = ((long)(A.N - n0) * A.L - l0) * 4;
        unsigned off[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) off[i] = l0 + 4 * (piece ^ (4 * i)) < A.L ? drow + 16u * (piece ^ (4 * i)) : (unsigned)ACT8_BEHIND;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(act8_rsrc(src, size), (act8_lds_t *)(mine + buf * BUF + i * 256), 16, off[i & 1], 0, 0, 0);
            src += eight;
            size -= eight * 4;
        }
    };
    bf16x8 a[2][3], w[2][4][3];
    Act8Codes<4> now, ahead;                                                 // a step's codes, the next one's
    auto rows_of = [&](int t, int j, int buf, bf16x8 (&o)[3], bool counts = true) __attribute__((always_inline)) {
        float va[8];
        const float *row = mine + buf * BUF + (32 * t + r) * 32;
        const int key = r >> 1 & 7;
        const f32x4 e0 = *reinterpret_cast<const f32x4 *>(row + ((4 * h + 2 * j) ^ key) * 4);
        const f32x4 e1 = *reinterpret_cast<const f32x4 *>(row + ((4 * h + 2 * j + 1) ^ key) * 4);
#pragma unroll
        for (int x = 0; x < 4; ++x) { va[x] = e0[x]; va[4 + x] = e1[x]; }
        const float sum = ((va[0] + va[1]) + (va[2] + va[3])) + ((va[4] + va[5]) + (va[6] + va[7]));
        db[t] += counts ? sum : 0.f;
        act8_split(va, o[0], o[1], o[2]);
    };
    auto operand_of = [&](const Act8Codes<4> &M, int t, int j, bf16x8 (&o)[3]) __attribute__((always_inline)) {
        const float cs = ga[t] * M.s[t];
        if (j == 0) poison[t] += cs * 0.f;
        act8_operand<NORM>(M.q[t], j, cs, be[t], M.m[t] >> (8 * h), flip, o);
    };
    if (first < A.steps) {
        Act8Step next = {first / turn.spc, first % turn.spc};                // behind the last step: the last one again
        act8_codes<4, NORM>(A, next, h, krow, now);
        dma(next, 0);
        if (first + stride < A.steps) next = turn.after(next);
        act8_codes<4, NORM>(A, next, h, krow, ahead);
        __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < 4; ++t) operand_of(now, t, 0, w[0][t]);
        rows_of(0, 0, 0, a[0]);
        int buf = 0;
#pragma unroll 1
        for (int s = first; s < A.steps; s += stride) {
            const bool more = s + stride < A.steps;
            dma(next, buf ^ 1);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    if (j == 1 && t == 3) {
                        __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));    // the next step's rows have arrived
                        asm volatile("" ::: "memory");
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    operand_of(j ? ahead : now, t, j ^ 1, w[j ^ 1][t]);
                    if (t < 3) rows_of(t + 1, j, buf, a[(t + 1) & 1]);
                    else if (j == 0) rows_of(0, 1, buf, a[0]);
                    else rows_of(0, 0, buf ^ 1, a[0], more);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int c = 0; c < 6; ++c) acc[t][k] = MFMAB(a[t & 1][act8_first(c)], w[j][k][act8_second(c)], acc[t][k]);
                    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);       // LDS reads
#pragma unroll
                    for (int i = 0; i < 24; ++i) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // a product
                        __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);   // vector instructions
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            now = ahead;
            if (s + 2 * stride < A.steps) next = turn.after(next);
            act8_codes<4, NORM>(A, next, h, krow, ahead);
            buf ^= 1;
        }
    }
    __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));                        // nothing may be on its way into LDS when the shares go there
    asm volatile("" ::: "memory");
    act8_wgrad_end<4, 4>(A, lds, acc, db, poison, flip, at.slice, n0, k0);
}

// Few channels (N <= 64, K <= 64): both products of the backward pass are bound by reading g, so one kernel makes them.  A wave keeps
// 32 RT x 32 of dW as above, and for the same 32 points W^T . g from the same piece of LDS (lane = point, its eight values of a
// k-step from eight rows), the fragments of W^T in LDS too.  dy goes to dx's place, its two sums stay in registers to the end.
// Either product alone comes from here too, so that it does not depend on what else is asked for.
// 32 -> 64 over 1,048,576 points: 103 to 111 us (118 before its g went past the caches) against 93 + 104 for the two, 64 -> 64 over 524,288:
// 109 against 52 + 78.
struct Act8Both {
    Act8Wgrad w;
    const float *W;
    float *dx;             // (B, K, L): dy
    float *part;           // NORM: {sum dy, sum dy*uh}[K][2][waves that share a tile]
};
template <int RT, bool NORM>
__global__ __launch_bounds__(256, 2) void p2n_act8_both_kernel(Act8Both B) {
    const Act8Wgrad &A = B.w;
    constexpr int BUF = RT * 4096;                                           // bytes; 32 RT rows of 32 points
    __shared__ __attribute__((aligned(16))) char lds[4 * BUF];
    __shared__ __attribute__((aligned(16))) char wt[RT * 6144];              // k-step, part: 1 KiB
    __shared__ __attribute__((aligned(16))) unsigned kept[NORM ? 4 : 1][320];       // the wave's: scales of its 32 channels, bits, codes (32 points a row)
    static_assert(4 * BUF >= act8_join_floats(RT, 1) * 4, "the shares pass through the same memory");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int r = lane & 31, h = lane >> 5;
    const Act8Place at = act8_place(A);
    const int k0 = at.tile * 32, turn = A.slices * 4, first = at.slice * 4 + wave;
    const Act8Turn take(A, turn);
    const unsigned flip = (unsigned)(first & 1) << 31;                       // every other wave has g with its sign turned round (act8_flip)
    for (int ks = wave; ks < 2 * RT; ks += 4) {
        const int k = k0 + r, n = 16 * ks + 8 * h;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = n + i < A.N && k < A.K ? B.W[(long)(n + i) * A.K + k] : 0.f;
        bf16x8 *d = reinterpret_cast<bf16x8 *>(wt + ks * 3 * 1024) + lane;
        act8_split_rounded(v, d[0], d[64], d[128]);
    }
    __syncthreads();
    const int krow = k0 + r < A.K ? k0 + r : A.K - 1;
    const float ga = NORM ? A.gamma[krow] : 1.f, be = NORM ? A.beta[krow] : 0.f;
    float poison[1] = {act8_poison<NORM>(be)}, db[RT], s1[16], s2[16];
    f32x16 acc[RT][1];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        db[i] = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][0][e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) s1[e] = s2[e] = 0.f;
    char *const mine = lds + wave * BUF;
    const int drow = lane >> 3, slot = (lane & 7) ^ (lane >> 4);
    int qn[4];
    float sn;
    unsigned mn;
    auto meta = [&](Act8Step s) __attribute__((always_inline)) {
        const long blk = s.b * A.NB + (s.q >> 2);
        const int w = s.q & 3;
        const i32x4 q = *reinterpret_cast<const i32x4 *>(A.codes + (blk * A.K + krow) * ACT8_GROUP + 32 * w + 16 * h);
#pragma unroll
        for (int x = 0; x < 4; ++x) qn[x] = q[x];
        sn = A.scale[blk * A.K4 + krow];
        mn = NORM ? A.bits[(blk * 4 + w) * A.K4 + krow] : 0u;
    };
    f32x4 vn[RT * 4];
    const bool full = A.N == 32 * RT;
    auto rows = [&](Act8Step s) __attribute__((always_inline)) {
        const long b = s.b, l0 = (long)s.q * 32, l = l0 + 4 * (lane & 7);
        const bool whole = full && l0 + 32 <= A.L;
#pragma unroll
        for (int i = 0; i < RT * 4; ++i) {
            const int n = 8 * i + drow;
            const float *p = A.g + (b * A.N + (n < A.N ? n : A.N - 1)) * A.L + l;
            if (whole) vn[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4u *>(p));
            else
#pragma unroll
                for (int x = 0; x < 4; ++x) vn[i][x] = n < A.N && l + x < A.L ? p[x] : 0.f;
        }
    };
    Act8Step step = {first / take.spc, first % take.spc};
    if (first < A.steps) {
        rows(step);
        meta(step);
    }
#pragma unroll 1
    for (int s = first; s < A.steps; s += turn) {
#pragma unroll
        for (int i = 0; i < RT * 4; ++i) {
            f32x4 v = vn[i];
#pragma unroll
            for (int x = 0; x < 4; ++x) v[x] = act8_flip(v[x], flip);
            *reinterpret_cast<f32x4 *>(mine + i * 1024 + drow * 128 + (slot ^ (4 * (i & 1))) * 16) = v;
        }
        int q[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) q[x] = qn[x];
        const float cs = ga * sn;
        poison[0] += cs * 0.f;                              // NaN with a NaN scale
        const unsigned mb = mn >> (8 * h);                  // points 16h .. 16h+15: bits 8h .. of either half-word
        if (NORM) {
            *reinterpret_cast<i32x4 *>(&kept[wave][64 + 8 * r + 4 * h]) = i32x4{q[0], q[1], q[2], q[3]};
            kept[wave][lane] = h ? mn : __float_as_uint(sn);
        }
        const Act8Step now = step;
        step = take.after(step);
        if (s + turn < A.steps) {
            rows(step);
            meta(step);
        }
        if (A.part) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                bf16x8 w[3];
                act8_operand<NORM>(i32x4{q[0], q[1], q[2], q[3]}, j, cs, be, mb, 0u, w);
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    float va[8];
                    const char *row = mine + (32 * t + r) * 128;
                    const int key = r >> 1 & 7;
                    const f32x4 e0 = *reinterpret_cast<const f32x4 *>(row + ((4 * h + 2 * j) ^ key) * 16);
                    const f32x4 e1 = *reinterpret_cast<const f32x4 *>(row + ((4 * h + 2 * j + 1) ^ key) * 16);
#pragma unroll
                    for (int x = 0; x < 4; ++x) { va[x] = e0[x]; va[4 + x] = e1[x]; }
                    if (k0 == 0) db[t] += ((va[0] + va[1]) + (va[2] + va[3])) + ((va[4] + va[5]) + (va[6] + va[7]));
                    bf16x8 a[3];
                    act8_split(va, a[0], a[1], a[2]);
#pragma unroll
                    for (int c = 0; c < 6; ++c) acc[t][0] = MFMAB(a[act8_first(c)], w[act8_second(c)], acc[t][0]);
                    if (t & 1) __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (!B.dx) continue;
        f32x16 da;
#pragma unroll
        for (int e = 0; e < 16; ++e) da[e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 2 * RT; ++ks) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[i] = *reinterpret_cast<const float *>(mine + (16 * ks + 8 * h + i) * 128 + ((r >> 2) ^ (4 * h + (i >> 1))) * 16 + (r & 3) * 4);
            bf16x8 xp[3];
            act8_split(x, xp[0], xp[1], xp[2]);
            const bf16x8 *f = reinterpret_cast<const bf16x8 *>(wt + ks * 3 * 1024) + lane;
#pragma unroll
            for (int c = 0; c < 6; ++c) da = MFMAB(f[64 * act8_first(c)], xp[act8_second(c)], da);
            if (ks & 1) __builtin_amdgcn_sched_barrier(0);
        }
        const long l = (long)now.q * 32 + r;
        const __amdgpu_buffer_rsrc_t ro = act8_rsrc(B.dx + ((long)now.b * A.K + k0) * A.L, (long)(A.K - k0) * A.L * 4);    // channels past K are not stored
        const unsigned oo = (unsigned)((4 * h * A.L + l) * 4);
        const int bit = (r >> 1) + 16 * (r & 1);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            i32x4 sc = {0, 0, 0, 0}, on = {0, 0, 0, 0};
            if (NORM) {
                sc = *reinterpret_cast<const i32x4 *>(&kept[wave][8 * g + 4 * h]);
                on = *reinterpret_cast<const i32x4 *>(&kept[wave][32 + 8 * g + 4 * h]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int e = 4 * g + j;
                float dy = act8_flip(da[e], flip);
                if (NORM) {
                    const bool above = on[j] >> bit & 1;
                    const int code = reinterpret_cast<const signed char *>(&kept[wave][64 + 8 * (8 * g + 4 * h + j)])[r];
                    dy = above ? dy : 0.f;
                    s1[e] += dy;
                    s2[e] += above ? dy * ((float)code * __int_as_float(sc[j])) : 0.f;
                }
                if (l < A.L) __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(dy), ro, oo + (unsigned)((8 * g + j) * A.L * 4), 0, 0);
            }
        }
    }
    if (NORM && B.dx) {
        const float t1 = act8_half_sum(s1, lane), t2 = act8_half_sum(s2, lane);
        const int i = lane & 15, k = k0 + 8 * (i >> 2) + 4 * h + (i & 3);
        if (!(lane & 16) && k < A.K) {
            B.part[((long)k * 2) * turn + first] = t1;
            B.part[((long)k * 2 + 1) * turn + first] = t2;
        }
    }
    if (!A.part) return;
#pragma unroll
    for (int t = 0; t < RT; ++t) db[t] = act8_flip(db[t], flip);
    act8_wgrad_end<RT, 1>(A, reinterpret_cast<float *>(lds), acc, db, poison, flip, at.slice, 0, k0);
}

// out[i] = sum over slices, in a fixed order: the slices dealt to R rows of threads, 1024 / R results a workgroup; R = 4 where there are
// few slices of so many results that the card is full (384 -> 256, 21 slices: 4.2 us against 8.7; 256 -> 256, 64: 8.8 against 9.5;
// with 67 -> 100, 26 workgroups to 209, it gains nothing).  The first n0 results are dW, the others db (either may be NULL).  The first split_wgs
// workgroups make the image of W^T.
template <int R>
__global__ __launch_bounds__(1024) void p2n_act8_join_kernel(const float *__restrict__ part, long n, long n0, int slices, float *__restrict__ dW, float *__restrict__ db,
                                                             Act8Split split, int split_wgs) {
    constexpr int W = 1024 / R;
    __shared__ float sh[R][W + 1];
    const int blk = (int)blockIdx.x - split_wgs;
    if (blk < 0) {
        act8_split_weights(split, (long)blockIdx.x * 1024 + threadIdx.x);
        return;
    }
    const int o = threadIdx.x % W, y = threadIdx.x / W;
    const long i = (long)blk * W + o;
    float s = 0.f;
    if (i < n)
        for (int k = y; k < slices; k += R) s += part[k * n + i];
    sh[y][o] = s;
    __syncthreads();
    if (y == 0 && i < n) {
        for (int k = 1; k < R; ++k) s += sh[k][o];
        if (i < n0) {
            if (dW) dW[i] = s;
        } else if (db) {
            db[i - n0] = s;
        }
    }
}

// ---------------------------------------------------------------- norm + ReLU alone (the end of a chain), backward
// dy = [y > 0] * g and its sums; one workgroup per (channel, slice of the (cloud, block) list), a wave takes a block, a lane two points
__global__ __launch_bounds__(256) void p2n_act8_dy_kernel(const float *__restrict__ g, int B, int C, int C4, long L, long NB, long per,
                                                          const signed char *__restrict__ codes, const float *__restrict__ scale, const unsigned *__restrict__ bits,
                                                          float *__restrict__ dy, float *__restrict__ part) {
    __shared__ float sh[8];
    const int c = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long n = (long)B * NB, i0 = (long)blockIdx.y * per, i1 = i0 + per < n ? i0 + per : n;
    float u = 0.f, v = 0.f;
    for (long i = i0 + wave; i < i1; i += 4) {
        const long b = i / NB, l = (i % NB) * ACT8_GROUP + 2 * lane, row = b * C + c;
        const float s = scale[i * C4 + c];
        const unsigned w = bits[(i * 4 + (lane >> 4)) * C4 + c];
        const int q = *reinterpret_cast<const unsigned short *>(codes + (i * C + c) * ACT8_GROUP + 2 * lane);
        if (l >= L) continue;
        const bool two = l + 1 < L, on0 = w >> (lane & 15) & 1, on1 = w >> (16 + (lane & 15)) & 1;
        f32x2 e = {0.f, 0.f};
        if (two) e = *reinterpret_cast<const f32x2u *>(g + row * L + l);
        else e[0] = g[row * L + l];
        e[0] = on0 ? e[0] : 0.f;
        e[1] = on1 ? e[1] : 0.f;
        if (two) *reinterpret_cast<f32x2u *>(dy + row * L + l) = e;
        else dy[row * L + l] = e[0];
        u += e[0] + e[1];
        if (on0) v += e[0] * ((float)(signed char)q * s);
        if (on1) v += e[1] * ((float)(signed char)(q >> 8) * s);
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
    int RT, CT, ntc, nt, slices;     // weight gradient: 32-row tiles of a wave, tiles, slices of the points
    long wsteps;
    int both, waves;                 // weight and data gradient in one kernel: 32-row tiles of a wave (0: no), waves that share a tile
};

// Channel tiles of a workgroup: all of them (the points are then read once), fewer where there are so few blocks of points that compute
// units would stay without one (384 -> 256 at 8,192 points, 64 blocks: 36 us with 8 tiles, 17 with 2).
int act8_tiles(int rows, long blocks) {
    int ct = rows <= 32 ? 1 : rows <= 64 ? 2 : rows <= 128 ? 4 : 8;
    while (ct > 1 && blocks * ((rows + 32 * ct - 1) / (32 * ct)) < 256) ct >>= 1;
    return ct;
}
int act8_ksteps(int k, int ct) {
    const int cks = act8_chunk(ct), ks = (k + 15) / 16;
    return (ks + cks - 1) / cks * cks;
}
int act8_padded(int rows, int ct) { return ((rows + 31) / 32 + ct - 1) / ct * ct; }

void act8_wgrad_tiles(Act8 &a, int rt, int ct) {
    a.RT = rt; a.CT = ct;
    a.ntc = (a.K + 32 * ct - 1) / (32 * ct);
    a.nt = ((a.N ? a.N : 1) + 32 * rt - 1) / (32 * rt) * a.ntc;
}

int act8_init(Act8 &a, const char *fn, int B, int K, long L, int N) {
    P2N_REQUIRE(B >= 1 && L >= 1 && L <= (1L << 24), "%s: bad shape B=%d L=%ld (1 to 2^24 columns a cloud)", fn, B, L);
    P2N_REQUIRE(K >= 1 && K <= ACT8_MAX_C && N >= 0 && N <= ACT8_MAX_C, "%s: %d or %d channels, not in [1,%d]", fn, K, N, ACT8_MAX_C);
    a.B = B; a.K = K; a.N = N; a.L = L; a.NB = (L + ACT8_GROUP - 1) / ACT8_GROUP;
    // a launch holds less than 2^32 threads: 2^24 workgroups of 256, of which the weight image takes up to 1024
    P2N_REQUIRE((long)B * a.NB <= (1L << 24) - 1025, "%s: too many points (%ld blocks of 128)", fn, (long)B * a.NB);
    a.Kpad = (K + 63) / 64 * 64;
    const int cf = act8_tiles(N ? N : 1, (long)B * a.NB), cb = act8_tiles(K, (long)B * a.NB);
    a.KSf = act8_ksteps(K, cf); a.CTf = act8_padded(N ? N : 1, cf);
    a.KSb = act8_ksteps(N ? N : 1, cb); a.CTb = act8_padded(K, cb);
    const long blocks = (long)B * ((L + 2047) / 2048);
    long s = 2048 / K > 1 ? 2048 / K : 1;
    if (s > blocks) s = blocks;
    if (s > 1024) s = 1024;
    if (blocks <= 4) s = 1;              // few enough for one workgroup a channel, which then needs no second kernel
    a.per = (blocks + s - 1) / s;
    a.S = (int)((blocks + a.per - 1) / a.per);
    // a wave makes up to 64 x 64, two of them on a SIMD; 128 x 128 (which fills the registers alone, and splits each operand half as
    // often) where both sides are that long and there are points enough for such waves: 256 x 256 at 131,072 points 127 us against
    // 155, 64 x 128 at 262,144 points 70 against 55 with 128 rows, 256 x 384 at 8,192 points 56 against 19
    a.wsteps = (long)B * a.NB * 4;
    const bool big = N >= 128 && K >= 128 && a.wsteps >= 2048 && L % 4 == 0;
    act8_wgrad_tiles(a, big ? 4 : N <= 32 ? 1 : 2, big ? 4 : K <= 32 ? 1 : 2);
    const long wgs = a.RT * a.CT >= 8 ? 256 : a.RT * a.CT >= 4 ? 512 : a.RT * a.CT == 2 ? 768 : 1024;
    long sl = wgs / a.nt > 1 ? wgs / a.nt : 1;
    if (sl > (a.wsteps + 7) / 8) sl = (a.wsteps + 7) / 8;
    a.slices = (int)sl;
    // both gradients in one kernel, two workgroups of four waves a compute unit, up to 64 x 64: beyond, a wave's sums and rows leave no
    // registers to overlap with (64 -> 128 over 262,144 points: 126 us against 46 + 49)
    a.both = N < 1 || N > 64 || K > 64 ? 0 : N <= 32 ? 1 : 2;
    a.waves = 0;
    if (a.both) {
        const long most = 2048 / ((K + 31) / 32);
        a.waves = (int)((most < a.wsteps ? most : a.wsteps) + 3) / 4 * 4;
    }
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
    float *part, *tab, *wpart;
    __bf16 *img;
    long nparts;
    size_t total;
};
BwdSpace bwd_space(const Act8 &a, char *base) {
    Carve c{base, 0};
    BwdSpace f;
    f.nparts = a.both ? a.waves : a.N ? (long)a.B * a.NB : a.S;
    f.part = c.take<float>((size_t)2 * a.K * f.nparts);
    f.tab = c.take<float>((size_t)3 * a.K);
    f.img = c.take<__bf16>(a.both ? 0 : (size_t)a.CTb * a.KSb * 1536);
    f.wpart = c.take<float>((size_t)(a.both ? a.waves / 4 : a.slices) * (a.N * (size_t)a.K + a.N));
    f.total = c.off;
    return f;
}

template <int IN, int EPI, int TABK>
int act8_launch_gemm_tab(const Act8Gemm &g, long groups, hipStream_t s) {
    const int ct = act8_tiles(g.rows, groups);
    const dim3 grid((unsigned)groups, (unsigned)(g.CTP / ct)), blk(256);
    switch (ct) {
        case 1: hipLaunchKernelGGL((p2n_act8_gemm_kernel<IN, EPI, 1, TABK>), grid, blk, 0, s, g); break;
        case 2: hipLaunchKernelGGL((p2n_act8_gemm_kernel<IN, EPI, 2, TABK>), grid, blk, 0, s, g); break;
        case 4: hipLaunchKernelGGL((p2n_act8_gemm_kernel<IN, EPI, 4, TABK>), grid, blk, 0, s, g); break;
        default: hipLaunchKernelGGL((p2n_act8_gemm_kernel<IN, EPI, 8, TABK>), grid, blk, 0, s, g);
    }
    P2N_CHECK_HIP(hipGetLastError());
    return P2N_OK;
}
template <int IN, int EPI>
int act8_launch_gemm(const Act8Gemm &g, long groups, hipStream_t s) {
    if constexpr (IN == ACT8_NORM)
        if (g.Kpad > 512) return act8_launch_gemm_tab<IN, EPI, ACT8_MAX_C>(g, groups, s);
    return act8_launch_gemm_tab<IN, EPI, 512>(g, groups, s);
}

template <bool NORM>
int act8_launch_wgrad(const Act8 &a, const Act8Wgrad &w, hipStream_t s) {
    const dim3 grid((unsigned)(a.nt * a.slices)), blk(256);
    if (a.RT == 4) hipLaunchKernelGGL(p2n_act8_wgrad_wide_kernel<NORM>, grid, blk, 0, s, w);
    else if (a.RT == 2 && a.CT == 2) hipLaunchKernelGGL((p2n_act8_wgrad_kernel<2, 2, NORM>), grid, blk, 0, s, w);
    else if (a.RT == 2) hipLaunchKernelGGL((p2n_act8_wgrad_kernel<2, 1, NORM>), grid, blk, 0, s, w);
    else hipLaunchKernelGGL((p2n_act8_wgrad_kernel<1, 2, NORM>), grid, blk, 0, s, w);      // N <= 32 means K > 64 here
    P2N_CHECK_HIP(hipGetLastError());
    return P2N_OK;
}

template <bool NORM>
int act8_launch_both(const Act8 &a, Act8Both &b, hipStream_t s) {
    b.w.slices = a.waves / 4;
    const dim3 grid((unsigned)((a.K + 31) / 32 * b.w.slices)), blk(256);
    if (a.both == 2) hipLaunchKernelGGL((p2n_act8_both_kernel<2, NORM>), grid, blk, 0, s, b);
    else hipLaunchKernelGGL((p2n_act8_both_kernel<1, NORM>), grid, blk, 0, s, b);
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

// statistics and tables of x (norm), and what is kept of it; relu(y) to `out`, or the image of `split`
int act8_keep(const Act8 &a, const float *x, const float *gamma, const float *beta, float *rmean, float *rvar, long *batches, float momentum, float eps,
              char *kept, const FwdSpace &f, float *out, const Act8Split &split, hipStream_t s) {
    const Act8Kept k = act8_kept(a.B, a.K, a.L, gamma != nullptr);
    float *stat = (float *)(kept + k.stat);
    if (gamma) {
        const bool frozen = momentum < 0.f;
        const Act8Norm n{x, gamma, beta, rmean, rvar, batches, (double)momentum, (double)eps, (double)a.B * a.L, frozen ? 1 : 0, a.K, a.Kpad, a.L, stat, f.tab};
        const long blocks = (long)a.B * ((a.L + 2047) / 2048);
        if (!frozen && a.S == 1) {
            hipLaunchKernelGGL(p2n_act8_stats_kernel<true>, dim3(a.Kpad), dim3(256), 0, s, x, a.B, a.K, a.L, blocks, a.per, f.part, n);
        } else {
            if (!frozen) {
                hipLaunchKernelGGL(p2n_act8_stats_kernel<false>, dim3(a.K, a.S), dim3(256), 0, s, x, a.B, a.K, a.L, blocks, a.per, f.part, n);
                P2N_CHECK_HIP(hipGetLastError());
            }
            hipLaunchKernelGGL(p2n_act8_norm_kernel, dim3(a.Kpad), dim3(64), 0, s, f.part, a.S, n);
        }
        P2N_CHECK_HIP(hipGetLastError());
    }
    const Act8Keep keep{x, stat, gamma, beta, (signed char *)kept, (float *)(kept + k.scale), (unsigned *)(kept + k.bits), out, a.L, a.NB,
                        ((long)split.CTP * split.KS + 3) / 4, a.K, (a.K + 3) / 4 * 4, split};
    const dim3 grid((unsigned)(keep.split_wgs + (long)a.B * a.NB), (unsigned)((a.K + 31) / 32));
    if (out) hipLaunchKernelGGL((p2n_act8_keep_kernel<true, true>), grid, dim3(256), 0, s, keep);
    else if (gamma) hipLaunchKernelGGL((p2n_act8_keep_kernel<true, false>), grid, dim3(256), 0, s, keep);
    else hipLaunchKernelGGL((p2n_act8_keep_kernel<false, false>), grid, dim3(256), 0, s, keep);
    P2N_CHECK_HIP(hipGetLastError());
    return P2N_OK;
}

// dy in dx's place -> dx, dgamma, dbeta
int act8_through_norm(const Act8 &a, float *dx, const Act8Sums &n, const signed char *codes, const float *scale, hipStream_t s) {
    const dim3 grid((unsigned)((long)a.B * a.NB), (unsigned)((a.K + 31) / 32));
    const int C4 = (a.K + 3) / 4 * 4;
    if (n.n <= ACT8_FEW) {
        hipLaunchKernelGGL(p2n_act8_dx_kernel<true>, grid, dim3(256), 0, s, dx, a.K, C4, a.L, a.NB, n, codes, scale);
    } else {
        hipLaunchKernelGGL(p2n_act8_sums_kernel, dim3(a.K), dim3(256), 0, s, n);
        P2N_CHECK_HIP(hipGetLastError());
        hipLaunchKernelGGL(p2n_act8_dx_kernel<false>, grid, dim3(256), 0, s, dx, a.K, C4, a.L, a.NB, n, codes, scale);
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
                                float *running_mean, float *running_var, long *batches, float momentum, float eps, float *h, void *kept, size_t kept_bytes,
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
    Act8Gemm g = {};
    TRY(act8_keep(a, x, gamma, beta, running_mean, running_var, batches, momentum, eps, (char *)kept, f, nullptr, Act8Split{W, f.img, N, K, 0, a.CTf, a.KSf}, s));
    g.x = x; g.img = f.img; g.tab = f.tab; g.bias = bias; g.out = h; g.L = L; g.NB = a.NB;
    g.K = K; g.Kpad = a.Kpad; g.KS = a.KSf; g.CTP = a.CTf; g.rows = N;
    const long groups = (long)B * a.NB;
    const bool once = (long)B * N * L * 4 >= ACT8_LAST_CACHE;
    if (gamma) TRY((once ? act8_launch_gemm<ACT8_NORM, ACT8_OUT_ONCE>(g, groups, s) : act8_launch_gemm<ACT8_NORM, ACT8_OUT>(g, groups, s)));
    else TRY((once ? act8_launch_gemm<ACT8_PLAIN, ACT8_OUT_ONCE>(g, groups, s) : act8_launch_gemm<ACT8_PLAIN, ACT8_OUT>(g, groups, s)));
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
    if (a.RT == 4 && ((uintptr_t)g & 15) != 0) act8_wgrad_tiles(a, 2, 2);      // the wide kernel takes 16 bytes at a time
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
    const int K4 = (K + 3) / 4 * 4;
    const bool want = dW || db;
    if (want || (dx && a.both)) {
        Act8Both w = {};
        w.w.g = g; w.w.codes = codes; w.w.scale = scale; w.w.bits = bits; w.w.gamma = gamma; w.w.beta = beta; w.w.part = want ? f.wpart : nullptr;
        w.w.L = L; w.w.NB = a.NB; w.w.steps = (int)a.wsteps; w.w.N = N; w.w.K = K; w.w.K4 = K4; w.w.ntc = a.ntc; w.w.slices = a.slices;
        w.W = W; w.dx = dx; w.part = f.part;
        if (a.both) {
            TRY(gamma ? act8_launch_both<true>(a, w, s) : act8_launch_both<false>(a, w, s));
        } else {
            TRY(gamma ? act8_launch_wgrad<true>(a, w.w, s) : act8_launch_wgrad<false>(a, w.w, s));
        }
    }
    if (want || (dx && !a.both)) {
        const Act8Split split = dx && !a.both ? Act8Split{W, f.img, K, N, 1, a.CTb, a.KSb} : Act8Split{};
        const long n = want ? (long)N * K + N : 0;
        const int split_wgs = (split.CTP * split.KS + 15) / 16;
        const int slices = a.both ? a.waves / 4 : a.slices;
        if (slices > 64 || n < 256 * 256) hipLaunchKernelGGL(p2n_act8_join_kernel<32>, dim3((unsigned)(split_wgs + (n + 31) / 32)), dim3(1024), 0, s, f.wpart, n, (long)N * K, slices,
                                            dW, db, split, split_wgs);
        else hipLaunchKernelGGL(p2n_act8_join_kernel<4>, dim3((unsigned)(split_wgs + (n + 255) / 256)), dim3(1024), 0, s, f.wpart, n, (long)N * K, slices,
                                dW, db, split, split_wgs);
        P2N_CHECK_HIP(hipGetLastError());
    }
    if (dx && !a.both) {
        Act8Gemm q = {};
        q.x = g; q.img = f.img; q.out = dx; q.codes = codes; q.scale = scale; q.bits = bits; q.part = f.part; q.L = L; q.NB = a.NB;
        q.K = N; q.Kpad = (N + 63) / 64 * 64; q.KS = a.KSb; q.CTP = a.CTb; q.rows = K; q.rows4 = K4;
        if (gamma) TRY((act8_launch_gemm<ACT8_PLAIN, ACT8_DY>(q, groups, s)));
        else TRY((act8_launch_gemm<ACT8_PLAIN, ACT8_OUT>(q, groups, s)));
    }
    if (dx && gamma) TRY(act8_through_norm(a, dx, Act8Sums{f.part, f.nparts, K, frozen ? 1 : 0, (double)B * L, gamma, stat, dgamma, dbeta, f.tab}, codes, scale, s));
    p2n_prof_end(ps, s);
    return P2N_OK;
}

extern "C" int p2n_act8_norm_relu_forward(const float *x, int B, int C, long L, const float *gamma, const float *beta, float *running_mean,
                                          float *running_var, long *batches, float momentum, float eps, float *out, void *kept, size_t kept_bytes,
                                          void *workspace, size_t workspace_bytes, void *stream_) {
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
    TRY(act8_keep(a, x, gamma, beta, running_mean, running_var, batches, momentum, eps, (char *)kept, f, out, Act8Split{}, s));
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
    const long n = (long)B * a.NB, per = (n + a.S - 1) / a.S;
    const int C4 = (C + 3) / 4 * 4;
    hipLaunchKernelGGL(p2n_act8_dy_kernel, dim3(C, a.S), dim3(256), 0, s, g, B, C, C4, L, a.NB, per, codes, scale, (const unsigned *)(kept + k.bits), dx, f.part);
    P2N_CHECK_HIP(hipGetLastError());
    TRY(act8_through_norm(a, dx, Act8Sums{f.part, f.nparts, C, frozen ? 1 : 0, (double)B * L, gamma, stat, dgamma, dbeta, f.tab}, codes, scale, s));
    p2n_prof_end(ps, s);
    return P2N_OK;
}
