// Products in 8-bit integers for gfx950 (MI355X), one scale for a token (a point) and one for an output channel:
//     (sx_t, qx_t) = 8-bit rule over the K values of token t        (sw_n, qw_n) = 8-bit rule over row n of W (N, K)
//     y[t][n] = fl(fl(fl(sum_k qx qw) * sw_n) * sx_t) + b_n, then ReLU if asked
// The sum is exact in int32 (K <= 65536 keeps it below 2^31); its conversion to float32 and the two products round once
// each.  The values between the layers of p2n_int8_mlp take the token's scale first, fl(fl(fl(sum) * sx_t) * sw_n) + b_n: they are put
// into 8 bits again, one step in them can move a code, and with it the results by a step of 8 bits, so there the order belongs to
// the definition (a result's last step is all that it moves elsewhere).  The reference has no 8-bit path (its layers are Conv1d, reference point2net.py:9-34): the formulas above are the
// specification.  Two operators share the weight image and the rule (p2n_q8.h):
//   p2n_int8_linear  rows of K values (tokens), float32 or bfloat16
//   p2n_int8_mlp     the layers of a shared MLP over the columns of (B, C, L), on chip from the input to the result
#include <type_traits>
#include "p2n_q8.h"

#define MFMA_I8(a, b, c) __builtin_amdgcn_mfma_i32_32x32x32_i8((a), (b), (c), 0, 0, 0)
#define INT8_MAX_K 65536
#define INT8_MAX_N 65536
#define INT8_MAX_LAYERS 8

// ---------------------------------------------------------------- weight image
// Fragment f = ct * KT + kt, 1 KiB: lane (row r = lane & 31, half h = lane >> 5) holds the 16 codes of channel 32ct + r whose
// k = 32kt + 8g + 4h + j sit at byte 4g + j -- the k order in which the 32 x 32 product leaves a tile of channels in the
// lanes of its points, so that one layer's output is the next one's operand without moving.  KT = ceil(K/32) rounded up
// to even; outside the real extent the codes are zero.  Behind the codes: scales[32 CT], bias[32 CT].
struct Int8Image {
    int CT, KT;
    size_t scale, bias, total;   // byte offsets, size
};

static Int8Image int8_image(int K, int N) {
    Int8Image I;
    I.CT = (N + 31) / 32;
    I.KT = ((K + 31) / 32 + 1) & ~1;
    I.scale = (size_t)I.CT * I.KT * 1024;
    I.bias = I.scale + sizeof(float) * 32 * I.CT;
    I.total = I.bias + sizeof(float) * 32 * I.CT;
    return I;
}

// one wave per channel: maximum, scale, codes.  A norm behind the product (gamma not NULL) is folded in: w s and (b - mean) s + beta
// with s = gamma / sqrt(var + eps), in 64 bits until s and the bias are float32.
struct Int8Norm {
    const float *gamma, *beta, *mean, *var;
    double eps;
};
__global__ __launch_bounds__(256) void p2n_int8_pack_kernel(const float *__restrict__ W, const float *__restrict__ bias, int K, int N,
                                                            int CT, int KT, char *__restrict__ img, float *__restrict__ scale,
                                                            float *__restrict__ bimg, Int8Norm B) {
    const int lane = threadIdx.x & 63;
    const int n = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (n >= 32 * CT) return;
    const float *w = W + (long)n * K;
    float fold = 1.f, t = 0.f;
    if (n < N) {
        if (bias) t = bias[n];
        if (B.gamma) {
            const double f = (double)B.gamma[n] / sqrt((double)B.var[n] + B.eps);
            fold = (float)f;
            t = (float)(((double)t - (double)B.mean[n]) * f + (double)B.beta[n]);
        }
    }
    unsigned am = 0;
    if (n < N)
        for (int k = lane; k < K; k += 64) {
            const unsigned b = p2n_absbits(w[k] * fold);
            am = b > am ? b : am;
        }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const unsigned o = (unsigned)__shfl_xor((int)am, m);
        am = o > am ? o : am;
    }
    const float s = p2n_q8_scale(am);
    const P2nQ8 Q = p2n_q8_make(s);
    if (lane == 0) {
        scale[n] = n < N ? s : 0.f;
        bimg[n] = t;
    }
    const int ct = n >> 5, r = n & 31;
    const bool bad = !(s == s);
    for (int k4 = lane; k4 < 8 * KT; k4 += 64) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = 4 * k4 + j;
            v[j] = (n < N && k < K) ? w[k] * fold : 0.f;
        }
        int c[1];
        p2n_q8_pack(v, Q, c);
        const int kt = k4 >> 3, d = k4 & 7;   // dword d of the tile: half d & 1, group d >> 1
        *reinterpret_cast<int *>(img + ((size_t)(ct * KT + kt) * 64 + 32 * (d & 1) + r) * 16 + 4 * (d >> 1)) = bad ? 0 : c[0];
    }
}

extern "C" long p2n_int8_weight_bytes(int K, int N) {
    if (K < 1 || K > INT8_MAX_K || N < 1 || N > INT8_MAX_N) return -1;
    return (long)int8_image(K, N).total;
}

extern "C" int p2n_int8_pack_weight(const float *W, const float *bias, int K, int N, const float *gamma, const float *beta, const float *mean,
                                    const float *var, double eps, void *image, void *stream_) {
    P2N_REQUIRE(K >= 1 && K <= INT8_MAX_K && N >= 1 && N <= INT8_MAX_N, "p2n_int8_pack_weight: K=%d or N=%d not in [1,%d]", K, N, INT8_MAX_K);
    P2N_REQUIRE(W && image, "p2n_int8_pack_weight: null pointer");
    P2N_REQUIRE(!gamma || (beta && mean && var && eps >= 0), "p2n_int8_pack_weight: a norm needs gamma, beta, mean, variance and eps >= 0");
    P2N_REQUIRE(((uintptr_t)image & 15) == 0, "p2n_int8_pack_weight: the image must be 16-byte aligned");
    const Int8Image I = int8_image(K, N);
    char *img = (char *)image;
    hipStream_t s = (hipStream_t)stream_;
    const int ps = p2n_prof_begin(P2N_K_INT8_PACK, s);
    hipLaunchKernelGGL(p2n_int8_pack_kernel, dim3(8 * I.CT), dim3(256), 0, s, W, bias, K, N, I.CT, I.KT, img, (float *)(img + I.scale),
                       (float *)(img + I.bias), Int8Norm{gamma, beta, mean, var, eps});
    p2n_prof_end(ps, s);
    P2N_CHECK_HIP(hipGetLastError());
    return P2N_OK;
}

// ---------------------------------------------------------------- tokens
__device__ __forceinline__ float int8_load(const float *p) { return *p; }
__device__ __forceinline__ float int8_load(const __bf16 *p) { return (float)*p; }

// rows of K values -> codes (T, K) in order and scales (T): one wave per token
template <typename TX>
__global__ __launch_bounds__(256) void p2n_quantize_tokens_kernel(const TX *__restrict__ x, long T, int K, long ld, signed char *__restrict__ codes,
                                                                  float *__restrict__ scale) {
    const int lane = threadIdx.x & 63;
    const long t = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= T) return;
    const TX *row = x + t * ld;
    unsigned am = 0;
    for (int k = lane; k < K; k += 64) {
        const unsigned b = p2n_absbits(int8_load(row + k));
        am = b > am ? b : am;
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const unsigned o = (unsigned)__shfl_xor((int)am, m);
        am = o > am ? o : am;
    }
    const float s = p2n_q8_scale(am);
    const P2nQ8 Q = p2n_q8_make(s);
    const bool bad = !(s == s);
    if (lane == 0) scale[t] = s;
    for (int k = lane; k < K; k += 64) codes[t * K + k] = bad ? 0 : (signed char)p2n_q8_decide(int8_load(row + k), Q);
}

// The 16 values of a token that one lane of a fragment holds: k = 32kt + 8g + 4h + j, g and j from 0 to 3.  f32: four 16-byte loads
// from any 4-byte address, bf16: four 8-byte loads (VEC: rows start on 4 bytes) or value by value.
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x4u __attribute__((ext_vector_type(4), aligned(4)));
template <bool VEC>
__device__ __forceinline__ void int8_chunk(const float *row, int K, int k, float (&v)[4]) {
    if (k + 4 <= K) {
        const f32x4u e = *reinterpret_cast<const f32x4u *>(row + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = e[j];
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = k + j < K ? row[k + j] : 0.f;
    }
}
template <bool VEC>
__device__ __forceinline__ void int8_chunk(const __bf16 *row, int K, int k, float (&v)[4]) {
    if (VEC && k + 4 <= K) {
        const bf16x4u e = *reinterpret_cast<const bf16x4u *>(row + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (float)e[j];
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = k + j < K ? (float)row[k + j] : 0.f;
    }
}

// One token into fragments by 1 << shift lanes: lane i of them takes half i & 1 of k-tiles i >> 1, (i >> 1) + (1 << shift - 1), ...;
// put(kt, h, codes) stores 16 bytes.  Up to HOLD such rounds stay in registers between the maximum and the codes, longer
// rows are read twice.  `across` takes the maximum over the waves of a token.  Returns the token's scale.
#define INT8_HOLD 4
template <bool VEC, typename TX, typename PUT, typename MAX>
__device__ __forceinline__ float int8_token(const TX *row, int K, int KT, int i, int shift, PUT put, MAX across) {
    const int h = i & 1, kstep = 1 << (shift - 1), rounds = (KT + kstep - 1) >> (shift - 1);
    float v[INT8_HOLD][16];
    unsigned am = 0;
#pragma unroll
    for (int n = 0; n < INT8_HOLD; ++n) {
        const int kt = n * kstep + (i >> 1);
        if (n < rounds) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                float e[4];
                int8_chunk<VEC>(row, K, 32 * kt + 8 * g + 4 * h, e);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[n][4 * g + j] = e[j];
            }
        }
    }
#pragma unroll
    for (int n = 0; n < INT8_HOLD; ++n)
        if (n < rounds) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const unsigned u = p2n_absbits(v[n][e]);
                am = u > am ? u : am;
            }
        }
    for (int n = INT8_HOLD; n < rounds; ++n) {
        const int kt = n * kstep + (i >> 1);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float e[4];
            int8_chunk<VEC>(row, K, 32 * kt + 8 * g + 4 * h, e);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned u = p2n_absbits(e[j]);
                am = u > am ? u : am;
            }
        }
    }
    for (int m = 1; m < 1 << shift && m < 64; m <<= 1) {
        const unsigned o = (unsigned)__shfl_xor((int)am, m);
        am = o > am ? o : am;
    }
    const float s = p2n_q8_scale(across(am));
    const P2nQ8 Q = p2n_q8_make(s);
#pragma unroll
    for (int n = 0; n < INT8_HOLD; ++n) {
        const int kt = n * kstep + (i >> 1);
        if (n < rounds) {
            int c[4];
            p2n_q8_pack(v[n], Q, c);
            if (kt < KT) put(kt, h, i32x4{c[0], c[1], c[2], c[3]});
        }
    }
    for (int n = INT8_HOLD; n < rounds; ++n) {
        const int kt = n * kstep + (i >> 1);
        float e[16];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float q[4];
            int8_chunk<VEC>(row, K, 32 * kt + 8 * g + 4 * h, q);
#pragma unroll
            for (int j = 0; j < 4; ++j) e[4 * g + j] = q[j];
        }
        int c[4];
        p2n_q8_pack(e, Q, c);
        if (kt < KT) put(kt, h, i32x4{c[0], c[1], c[2], c[3]});
    }
    return s;
}

// Tokens into fragments: tile tt of 32 tokens, fragment tt * KT + kt laid out as in the weight image; scales (32 TT).  16384 x 2048
// bfloat16: 38 us, 2.7 TB/s; memory alone would take 20, vector instructions fill half of the issue slots.  The rows behind
// the last token of a tile are left as they are: what they give is not stored.
template <typename TX, bool VEC>
__global__ __launch_bounds__(256) void p2n_int8_tile_kernel(const TX *__restrict__ x, long T, int K, long ld, int KT, int shift, char *__restrict__ img,
                                                            float *__restrict__ scale) {
    __shared__ unsigned sh[4];
    const long t = ((long)blockIdx.x * 256 + threadIdx.x) >> shift;
    const int i = threadIdx.x & ((1 << shift) - 1);
    const bool real = t < T;                                   // every lane stays: the maximum is taken over whole waves
    char *dst = img + ((t >> 5) * KT * 64 + (t & 31)) * 16;
    const float s = int8_token<VEC>(x + (real ? t : T - 1) * ld, K, KT, i, shift, [&](int kt, int h, i32x4 c) {
        if (real) *reinterpret_cast<i32x4 *>(dst + ((long)kt * 64 + 32 * h) * 16) = c;
    }, [&](unsigned am) {
        if (shift <= 6) return am;
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = am;
        __syncthreads();
        const int w0 = shift == 7 ? (threadIdx.x >> 7) * 2 : 0;
        unsigned m = sh[w0] > sh[w0 + 1] ? sh[w0] : sh[w0 + 1];
        if (shift == 8) {
            const unsigned o = sh[2] > sh[3] ? sh[2] : sh[3];
            m = o > m ? o : m;
        }
        return m;
    });
    if (real && i == 0) scale[t] = s;
}

__device__ __forceinline__ void int8_store(float *p, float v) { *p = v; }
__device__ __forceinline__ void int8_store(__bf16 *p, float v) { *p = (__bf16)v; }

__device__ __forceinline__ float int8_value(int acc, float sx, float sw, float b, int relu) {
    const float v = (float)acc * sw * sx + b;   // the token's scale last: it may be as large as float32 goes
    return relu && v <= 0.f ? 0.f : v;   // a NaN stays
}

// ---------------------------------------------------------------- product of fragments
// D = X . W^T, registers = tokens, lane = channel.  WR x WC waves of 32 TM tokens x 32 TN channels each.  Both operands
// pass through LDS by DMA, 64 values of k at a time, in a ring of RING; a read of the next fragments is always on its
// way while the matrix cores work on the present ones.  The largest tile is 128 x 256 by four waves, two workgroups on a compute unit: the
// LDS then carries 288 cycles of traffic to 256 of products, and one workgroup's output goes on beside the other's products
// (16384 x 2048 x 4096: 161 us, 1.7 POP/s; 256 x 256 by eight waves alone on a compute unit 166, by four waves 220).
typedef __attribute__((address_space(3))) void int8_lds_t;

// a tile's results to memory: lane = channel n, v[j] = token t + j
__device__ __forceinline__ void int8_store4(float *y, long t, long T, int N, int n, bool col, const float (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (col && t + j < T) y[(t + j) * N + n] = v[j];
}
// bfloat16: neighbouring lanes exchange, an even lane stores two channels of tokens t and t + 2, an odd one of t + 1 and t + 3, so that a
// store is a whole dword.  Only where rows start on 4 bytes (N even) and both channels are real.
__device__ __forceinline__ void int8_store4(__bf16 *y, long t, long T, int N, int n, bool col, const float (&v)[4]) {
    if (N & 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (col && t + j < T) y[(t + j) * N + n] = (__bf16)v[j];
        return;
    }
    const bool odd = n & 1;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const float keep = odd ? v[2 * p + 1] : v[2 * p], give = odd ? v[2 * p] : v[2 * p + 1];
        const float got = __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(give), 0xB1, 0xF, 0xF, true));   // lane ^ 1
        __bf16 two[2];
        two[0] = (__bf16)(odd ? got : keep);
        two[1] = (__bf16)(odd ? keep : got);
        const long tt = t + 2 * p + (odd ? 1 : 0);
        if (col && tt < T) *reinterpret_cast<unsigned *>(y + tt * N + (n & ~1)) = *reinterpret_cast<const unsigned *>(two);
    }
}

template <typename TY, int TM, int TN, int WR, int WC, int RING>
__global__ __launch_bounds__(64 * WR * WC, TM * TN >= 4 ? 2 : 4) void p2n_int8_gemm_kernel(const char *__restrict__ xi, const float *__restrict__ sx,
                                                                                          const char *__restrict__ wi, const float *__restrict__ sw,
                                                                                          const float *__restrict__ bias, long T, int N, long TT, int CT, int KT,
                                                                                          int relu, int gx, long tiles, TY *__restrict__ y) {
    constexpr int TILES = WR * TM + WC * TN, TPW = TILES / (WR * WC);       // 32-row tiles of both operands; fetched by a wave
    static_assert(TPW * WR * WC == TILES, "every wave fetches the same number of tiles");
    constexpr int STAGE = TILES * 2048;               // two k-tiles each
    constexpr int GROUP = 2 * TPW;                    // DMA instructions of a wave and stage
    __shared__ __attribute__((aligned(16))) char ring[RING * STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int r = lane & 31, h = lane >> 5;
    // neighbouring workgroups go to the eight dies in turn: each die takes a part of the tiles, in bands of 4 rows, so that what its
    // L2 holds is used by several workgroups (16384 x 2048 x 4096: bands of 1: 170 us, of 4: 161, of 8: 209)
    const long per = (tiles + 7) / 8, id = (long)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (id >= tiles) return;
    const long gy = tiles / gx, band = id / (4L * gx), rows = gy - 4 * band < 4 ? gy - 4 * band : 4, in = id - band * 4 * gx;
    const long t0 = (4 * band + in % rows) * WR * TM;
    const int c0 = (int)(in / rows) * WC * TN;
    const int ns = KT / 2;                            // stages (KT is even)
    const char *src[TPW];                             // tiles past the last one fetch that
#pragma unroll
    for (int i = 0; i < TPW; ++i) {
        const int tile = wave * TPW + i, ch = tile - WR * TM;
        const long at = tile < WR * TM ? (t0 + tile < TT ? t0 + tile : TT - 1) : (c0 + ch < CT ? c0 + ch : CT - 1);
        src[i] = (tile < WR * TM ? xi : wi) + at * KT * 1024;
    }
    auto stage = [&](int s, int slot) __attribute__((always_inline)) {
        const int k = s < ns ? s : ns - 1;            // past the end the last stage again: the count of outstanding loads stays the same
#pragma unroll
        for (int i = 0; i < TPW; ++i) {
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(src[i]), 0, KT * 1024, 0x00020000);
            char *dst = ring + slot * STAGE + (wave * TPW + i) * 2048;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (int8_lds_t *)dst, 16, lane * 16, k * 2048, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (int8_lds_t *)(dst + 1024), 16, lane * 16, k * 2048 + 1024, 0, 0);
        }
    };
    const int wr = wave / WC, wc = wave % WC;
    i32x4 fa[2][TM], fb[2][TN];
    auto read = [&](int slot, int kt, i32x4 (&a)[TM], i32x4 (&b)[TN]) __attribute__((always_inline)) {
        const char *base = ring + slot * STAGE + kt * 1024 + lane * 16;
#pragma unroll
        for (int i = 0; i < TM; ++i) a[i] = *reinterpret_cast<const i32x4 *>(base + (wr * TM + i) * 2048);
#pragma unroll
        for (int i = 0; i < TN; ++i) b[i] = *reinterpret_cast<const i32x4 *>(base + (WR * TM + wc * TN + i) * 2048);
    };
    i32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int c = 0; c < TN; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][c][e] = 0;
#pragma unroll
    for (int s = 0; s < RING; ++s) {
        stage(s, s);
        __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_waitcnt((((RING - 1) * GROUP) & 15) | (7 << 4) | ((((RING - 1) * GROUP) >> 4) << 14));       // stage 0 has arrived
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(0, 0, fa[0], fb[0]);
#pragma unroll 1
    for (int s = 0, slot = 0; s < ns; ++s) {
        __builtin_amdgcn_sched_barrier(0);
        read(slot, 1, fa[1], fb[1]);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int c = 0; c < TN; ++c) acc[i][c] = MFMA_I8(fa[0][i], fb[0][c], acc[i][c]);
        __builtin_amdgcn_sched_barrier(0);
        // stage s+1 has arrived everywhere, and every wave has read the last of stage s, whose place stage s + RING takes
        __builtin_amdgcn_s_waitcnt((((RING - 2) * GROUP) & 15) | (7 << 4) | (0 << 8) | ((((RING - 2) * GROUP) >> 4) << 14));
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        stage(s + RING, slot);
        slot = slot == RING - 1 ? 0 : slot + 1;
        read(slot, 0, fa[0], fb[0]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int c = 0; c < TN; ++c) acc[i][c] = MFMA_I8(fa[1][i], fb[1][c], acc[i][c]);
    }
    __builtin_amdgcn_s_waitcnt(7 << 4);               // nothing may be on its way into LDS when the workgroup ends
    asm volatile("" ::: "memory");
#pragma unroll
    for (int c = 0; c < TN; ++c) {
        const int n = 32 * (c0 + wc * TN + c) + r;
        const bool col = n < N;
        const float w = col ? sw[n] : 0.f, b = col ? bias[n] : 0.f;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const long t = 32L * (t0 + wr * TM + i) + 8 * g + 4 * h;
                const bool some = t < T;                                          // (a lane stays for its neighbour's exchange)
                const f32x4 s4 = *reinterpret_cast<const f32x4 *>(sx + (some ? t : 0));      // the scales of a tile are 32, written or not
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = int8_value(acc[i][c][4 * g + j], s4[j], w, b, relu);
                int8_store4(y, t, T, N, n, col, v);
            }
    }
}

// ---------------------------------------------------------------- few tokens
// Up to 16 TT tokens: the weights' way from memory is the time, so a workgroup takes 16 channels and its eight waves share the length
// K, each streaming its part of the weights straight from memory into 16 x 16 x 64 products; the eight sums meet in LDS
// (whole numbers: any order; 16 tokens x 4096 x 4096: 6.5 us, 2.6 TB/s of weights).  OWN: up to 8 tokens of up to 4096 values are put
// into 8 bits here, a wave a token, into LDS; otherwise the tokens' fragments come from p2n_int8_tile_kernel.
#define MFMA_I8_16(a, b, c) __builtin_amdgcn_mfma_i32_16x16x64_i8((a), (b), (c), 0, 0, 0)
#define INT8_OWN_K 4096
template <typename TX, int TT, bool OWN, bool VEC>
__global__ __launch_bounds__(512) void p2n_int8_few_kernel(const TX *__restrict__ x, int T, int K, long ld, const char *__restrict__ xi, const float *__restrict__ sx,
                                                           const char *__restrict__ wi, const float *__restrict__ sw, const float *__restrict__ bias, int N,
                                                           int KT, int relu, TX *__restrict__ y) {
    __shared__ __attribute__((aligned(16))) char own[OWN ? 8 * INT8_OWN_K : 16];      // [k-tile][half][8 tokens][16 codes]
    __shared__ float ssx[16 * TT];
    __shared__ int red[8][TT][256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int r = lane & 15, q = lane >> 4;           // operand lane: row r, 16 codes of k-tile 2kb + (q >> 1), half q & 1
    const int c0 = blockIdx.x * 16;
    const char *wb = wi + ((long)(c0 >> 5) * KT * 64 + (q >> 1) * 64 + (q & 1) * 32 + (c0 & 16) + r) * 16;
    const int nb = KT / 2;
    constexpr int AHEAD = 8;                          // k-blocks of a wave whose weights are on their way at once
    i32x4 w[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
        const int kb = wave + 8 * i;
        w[i] = *reinterpret_cast<const i32x4 *>(wb + (long)(kb < nb ? kb : 0) * 2048);
    }
    if (OWN) {
        if (wave < T) {
            const float s = int8_token<VEC>(x + (long)wave * ld, K, KT, lane, 6, [&](int kt, int h, i32x4 c) {
                *reinterpret_cast<i32x4 *>(own + ((kt * 2 + h) * 8 + wave) * 16) = c;
            }, [](unsigned am) { return am; });
            if (lane == 0) ssx[wave] = s;
        }
    } else if ((int)threadIdx.x < 16 * TT) {
        ssx[threadIdx.x] = (int)threadIdx.x < T ? sx[threadIdx.x] : 0.f;
    }
    if (OWN) __syncthreads();
    i32x4 acc[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[t] = i32x4{0, 0, 0, 0};
    for (int k0 = wave; k0 < nb; k0 += 8 * AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int kb = k0 + 8 * i;
            if (kb < nb) {
#pragma unroll
                for (int t = 0; t < TT; ++t) {
                    i32x4 a;
                    if (OWN) a = *reinterpret_cast<const i32x4 *>(own + (((2 * kb + (q >> 1)) * 2 + (q & 1)) * 8 + (r & 7)) * 16);
                    else a = *reinterpret_cast<const i32x4 *>(xi + (((long)(t >> 1) * KT + 2 * kb + (q >> 1)) * 64 + (q & 1) * 32 + 16 * (t & 1) + r) * 16);
                    acc[t] = MFMA_I8_16(a, w[i], acc[t]);
                }
            }
            const int kn = kb + 8 * AHEAD;
            if (kn < nb) w[i] = *reinterpret_cast<const i32x4 *>(wb + (long)kn * 2048);
        }
    }
    // D: column = lane & 15 (channel), row = 4 (lane >> 4) + register (token)
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[wave][t][(4 * q + e) * 16 + r] = acc[t][e];
    __syncthreads();
    for (int i = threadIdx.x; i < TT * 256; i += 512) {
        const int t = i >> 4, n = c0 + (i & 15);
        if (t >= T || n >= N) continue;
        int sum = 0;
#pragma unroll
        for (int v = 0; v < 8; ++v) sum += red[v][i >> 8][i & 255];
        int8_store(y + (long)t * N + n, int8_value(sum, ssx[t], sw[n], bias[n], relu));
    }
}

static size_t int8_tiles_bytes(long T, int K) {
    const long TT = (T + 31) / 32, KT = ((K + 31) / 32 + 1) & ~1;
    return (size_t)TT * KT * 1024 + sizeof(float) * 32 * TT;
}

extern "C" int p2n_quantize_tokens(const void *x, int bf16, long T, int K, long ld, signed char *codes, float *scale, void *stream_) {
    P2N_REQUIRE(T >= 0 && T < (1L << 31) && K >= 1 && K <= INT8_MAX_K && ld >= K, "p2n_quantize_tokens: bad shape T=%ld K=%d ld=%ld", T, K, ld);
    if (T == 0) return P2N_OK;
    P2N_REQUIRE(x && codes && scale, "p2n_quantize_tokens: null pointer");
    hipStream_t s = (hipStream_t)stream_;
    const int ps = p2n_prof_begin(P2N_K_INT8_TOKENS, s);
    for (long t = 0; t < T; t += 1L << 25) {              // a launch holds less than 2^32 threads
        const long n = T - t < (1L << 25) ? T - t : 1L << 25;
        const dim3 grid((unsigned)((n + 3) / 4)), blk(256);
        if (bf16) hipLaunchKernelGGL(p2n_quantize_tokens_kernel<__bf16>, grid, blk, 0, s, (const __bf16 *)x + t * ld, n, K, ld, codes + t * K, scale + t);
        else hipLaunchKernelGGL(p2n_quantize_tokens_kernel<float>, grid, blk, 0, s, (const float *)x + t * ld, n, K, ld, codes + t * K, scale + t);
        P2N_CHECK_HIP(hipGetLastError());
    }
    p2n_prof_end(ps, s);
    return P2N_OK;
}

// Which kernel: up to 64 tokens the one that streams the weights once (16 tokens x 4096 x 4096: 7 us against 13 with 64 x 64 tiles), and
// of these up to 8 tokens of up to 4096 values put into 8 bits on the way: one launch instead of two (one token of 512 values 4.5 us
// against 4 + 3; 8 of 4096 12 against 4.5 + 6.8; 16 of 4096 19.5 against 4.7 + 6.5).
static bool int8_is_few(long T) { return T <= 64; }
static bool int8_is_own(long T, int K) { return T <= 8 && K <= INT8_OWN_K; }

extern "C" size_t p2n_int8_linear_workspace_bytes(long T, int K, int N) {
    if (T < 1 || T > (1L << 30) || K < 1 || K > INT8_MAX_K || N < 1 || N > INT8_MAX_N) return 0;
    return int8_is_own(T, K) ? 0 : int8_tiles_bytes(T, K);
}

template <typename TX, bool VEC>
static void int8_launch_few(const TX *x, int T, int K, long ld, const char *ws, const float *sx, const char *img, int N, int relu, TX *y, hipStream_t s) {
    const Int8Image I = int8_image(K, N);
    const float *sw = (const float *)(img + I.scale), *b = (const float *)(img + I.bias);
    const dim3 grid((unsigned)((N + 15) / 16)), blk(512);
    if (int8_is_own(T, K)) hipLaunchKernelGGL((p2n_int8_few_kernel<TX, 1, true, VEC>), grid, blk, 0, s, x, T, K, ld, nullptr, nullptr, img, sw, b, N, I.KT, relu, y);
    else if (T <= 16) hipLaunchKernelGGL((p2n_int8_few_kernel<TX, 1, false, VEC>), grid, blk, 0, s, x, T, K, ld, ws, sx, img, sw, b, N, I.KT, relu, y);
    else if (T <= 32) hipLaunchKernelGGL((p2n_int8_few_kernel<TX, 2, false, VEC>), grid, blk, 0, s, x, T, K, ld, ws, sx, img, sw, b, N, I.KT, relu, y);
    else hipLaunchKernelGGL((p2n_int8_few_kernel<TX, 4, false, VEC>), grid, blk, 0, s, x, T, K, ld, ws, sx, img, sw, b, N, I.KT, relu, y);
}

template <typename TX, int TM, int TN, int WR, int WC, int RING>
static void int8_launch_gemm(const char *ws, const float *sx, const char *img, const Int8Image &I, long T, int N, int relu, TX *y, hipStream_t s) {
    const long TT = (T + 31) / 32, gy = (TT + WR * TM - 1) / (WR * TM);
    const int gx = (I.CT + WC * TN - 1) / (WC * TN);
    const long tiles = gx * gy;
    hipLaunchKernelGGL((p2n_int8_gemm_kernel<TX, TM, TN, WR, WC, RING>), dim3((unsigned)((tiles + 7) / 8 * 8)), dim3(64 * WR * WC), 0, s, ws, sx, img,
                       (const float *)(img + I.scale), (const float *)(img + I.bias), T, N, TT, I.CT, I.KT, relu, gx, tiles, y);
}

template <typename TX, bool VEC>
static int int8_linear_run(const TX *x, long T, int K, long ld, const char *img, int N, int relu, TX *y, char *ws, hipStream_t s) {
    const Int8Image I = int8_image(K, N);
    const long TT = (T + 31) / 32;
    float *sx = (float *)(ws + (size_t)TT * I.KT * 1024);
    if (!int8_is_own(T, K)) {
        // lanes of a token: 64 values each (the reductions and divisions of a token cost as much as some 20 of them), fewer where that
        // leaves the card empty: below 2048 threads a compute unit, down to 16 values, at most four waves
        int shift = 1;
        while (shift < 8 && (1 << shift) * INT8_HOLD < 2 * I.KT) ++shift;
        while (shift < 8 && (1 << shift) < 2 * I.KT && (T << shift) < 256 * 2048) ++shift;
        hipLaunchKernelGGL((p2n_int8_tile_kernel<TX, VEC>), dim3((unsigned)(((T << shift) + 255) / 256)), dim3(256), 0, s, x, T, K, ld, I.KT, shift, ws, sx);
        P2N_CHECK_HIP(hipGetLastError());
    }
    if (int8_is_few(T)) {
        int8_launch_few<TX, VEC>(x, (int)T, K, ld, ws, sx, img, N, relu, y, s);
    } else {
        // the largest tile that still fills the 256 compute units, 128 x 256 with two workgroups each: larger tiles read less, fewer of
        // them leave compute units idle (K = 2048, N = 4096: T = 2048 30 us against 26 with 128 x 128, T = 4096 45 against 46)
        auto tiles = [&](int rows, int cols) { return ((TT + rows - 1) / rows) * ((I.CT + cols - 1) / cols); };
        if (tiles(4, 8) >= 512) int8_launch_gemm<TX, 2, 4, 2, 2, 3>(ws, sx, img, I, T, N, relu, y, s);
        else if (tiles(4, 4) >= 256) int8_launch_gemm<TX, 2, 2, 2, 2, 4>(ws, sx, img, I, T, N, relu, y, s);
        else int8_launch_gemm<TX, 1, 1, 2, 2, 4>(ws, sx, img, I, T, N, relu, y, s);
    }
    P2N_CHECK_HIP(hipGetLastError());
    return P2N_OK;
}

extern "C" int p2n_int8_linear(const void *x, int bf16, long T, int K, long ld, const void *image, int N, int relu, void *y, void *workspace,
                               size_t workspace_bytes, void *stream_) {
    P2N_REQUIRE(T >= 0 && T <= (1L << 30) && K >= 1 && K <= INT8_MAX_K && N >= 1 && N <= INT8_MAX_N && ld >= K,
                "p2n_int8_linear: bad shape T=%ld K=%d N=%d ld=%ld", T, K, N, ld);
    if (T == 0) return P2N_OK;
    P2N_REQUIRE(x && image && y, "p2n_int8_linear: null pointer");
    const size_t need = p2n_int8_linear_workspace_bytes(T, K, N);
    if (need && (!workspace || workspace_bytes < need)) {
        p2n_set_error("p2n_int8_linear: workspace %zu bytes < required %zu", workspace_bytes, need);
        return P2N_EWORKSPACE;
    }
    P2N_REQUIRE((((uintptr_t)workspace | (uintptr_t)image) & 15) == 0, "p2n_int8_linear: workspace and image must be 16-byte aligned");
    P2N_REQUIRE(((uintptr_t)x & (bf16 ? 1 : 3)) == 0, "p2n_int8_linear: x must be aligned to its type");
    P2N_REQUIRE(((uintptr_t)y & (bf16 && (N & 1) ? 1 : 3)) == 0, "p2n_int8_linear: y must start on 4 bytes (bfloat16 rows of an odd length: on 2)");
    hipStream_t s = (hipStream_t)stream_;
    const int ps = p2n_prof_begin(P2N_K_INT8_GEMM, s);
    const bool vec = ld % 2 == 0 && ((uintptr_t)x & 3) == 0;        // bfloat16 rows that start on 4 bytes
    const char *img = (const char *)image;
    char *ws = (char *)workspace;
    const int rc = !bf16 ? int8_linear_run<float, true>((const float *)x, T, K, ld, img, N, relu, (float *)y, ws, s)
                   : vec ? int8_linear_run<__bf16, true>((const __bf16 *)x, T, K, ld, img, N, relu, (__bf16 *)y, ws, s)
                         : int8_linear_run<__bf16, false>((const __bf16 *)x, T, K, ld, img, N, relu, (__bf16 *)y, ws, s);
    p2n_prof_end(ps, s);
    return rc;
}

// ---------------------------------------------------------------- shared MLP, on chip
// Lane = point, registers = channels (D = W . X), 32 points at a time through every layer.  The 32 x 32 product leaves
// channel 32ct + 8g + 4h + j of a lane's point in register 4g + j of its half h; four neighbours packed to a dword are the
// operand of the next layer in the k order of the weight image: nothing moves between lanes.
struct MlpLayer {
    const char *img;
    const float *scale, *bias;
    int KT, KTI, CT, N;   // k-tiles that hold channels, k-tiles in the image, channel tiles, channels
};
struct Int8MlpArgs {
    const float *x;   // (B, C, L)
    float *out;       // (B, N, L) or (B, N, L / group)
    long L, tiles, total;   // tiles per cloud, in all
    int C, nl, last_relu, group;
    MlpLayer layer[INT8_MAX_LAYERS];
};

// order-preserving image of a float for a signed maximum; every NaN on top
__device__ __forceinline__ int int8_key(float v) {
    const int b = __float_as_int(v);
    return v != v ? 0x7FFFFFFF : b ^ ((b >> 31) & 0x7FFFFFFF);
}
__device__ __forceinline__ int int8_unkey(int k) { return k ^ ((k >> 31) & 0x7FFFFFFF); }

// The 16 channels 32kt + 8g + 4h + j of this lane's point; `off` is the lane's byte offset (half's rows and column).  The resource
// starts at row 32kt and ends with the cloud's last row.  In a whole tile the rows' offsets are scalar operands; in the last one
// of a ragged C they are part of the lane's offset, which the resource's end is checked against (it is not checked with the scalar
// one): channels past C read as zero, and groups of eight that hold none are not read.
__device__ __forceinline__ void int8_mlp_load(const float *xb, long L, int C, int kt, unsigned off, float (&v)[16]) {
    const int real = C - 32 * kt;
    const long left = (long)real * L * 4;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(xb + 32L * kt * L), 0,
                                                                         (int)(left < 0xFFFFFFFFL ? left : 0xFFFFFFFFL), 0x00020000);
    if (real >= 32) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            v[e] = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, off, (int)((8 * (e >> 2) + (e & 3)) * L * 4), 0));
    } else {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            if (8 * g < real) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    v[4 * g + j] = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, off + (unsigned)((8 * g + j) * L * 4), 0, 0));
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * g + j] = 0.f;
            }
        }
    }
}

// A tile's values y to memory: channel tile ct of cloud b, columns of the wave's 32 points
__device__ __forceinline__ void int8_mlp_out(const Int8MlpArgs &A, int N, long b, bool valid, unsigned off, int ct, const float (&y)[16]) {
    // the resource starts at row 32ct and ends with the cloud's last row: channels past N are not written
    const long left = (long)(N - 32 * ct) * A.L * 4;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(A.out + (b * N + 32L * ct) * A.L, 0,
                                                                         (int)(left < 0xFFFFFFFFL ? left : 0xFFFFFFFFL), 0x00020000);
    if (valid && 32 * ct + 32 <= N) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(y[e]), rs, off, (int)((8 * (e >> 2) + (e & 3)) * A.L * 4), 0);
    } else if (valid) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(y[e]), rs, off + (unsigned)((8 * (e >> 2) + (e & 3)) * A.L * 4), 0, 0);
    }
}

__device__ __forceinline__ float int8_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }   // a NaN stays

// The last layer before a maximum over groups, its operands the other way round: lane = channel, acc[e] = point 8(e>>2) + 4h + (e&3), so that
// the maximum is formed in registers; ps: the scales of the 32 points.  Rounding keeps the order, so bias and ReLU follow the maximum, once
// (under a bias of +inf it is the smallest value that shows: -inf makes a NaN, anything else +inf).
// l0: the tile's first column.
__device__ __forceinline__ void int8_mlp_groups(const Int8MlpArgs &A, const MlpLayer &Y, int ct, const i32x16 &acc, const float *ps, long b, long l0, int lane) {
    const int p = lane & 31, h = lane >> 5;
    const float bi = Y.bias[32 * ct + p], turn = bi == __builtin_inff() ? -1.f : 1.f, sc = Y.scale[32 * ct + p] * turn;
    float m[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const f32x4 s = *reinterpret_cast<const f32x4 *>(ps + 8 * g + 4 * h);
        float t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = (float)acc[4 * g + j] * sc * s[j];
        m[g] = int8_max(int8_max(int8_max(t[0], t[1]), t[2]), t[3]);
    }
    // the halves of the wave hold every other four points: one exchange joins them, 16 points' maximum (32: both the same) to either half
    float u = int8_max(m[0], m[1]), w = int8_max(m[2], m[3]);
    if (A.group == 32) u = w = int8_max(u, w);
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_int(u), __float_as_int(w), false, false);
    float y = int8_max(__int_as_float(x[0]), __int_as_float(x[1])) * turn + bi;
    if (A.last_relu) y = y <= 0.f ? 0.f : y;
    const bool two = A.group == 16;
    if (32 * ct + p < Y.N && (two ? l0 + 16 * h < A.L : h == 0)) A.out[(b * Y.N + 32 * ct + p) * (A.L / A.group) + (two ? l0 / 16 + h : l0 / 32)] = y;
}

// A tile's sums to its values: scales, bias, ReLU; into `am` the largest of them as bits, where a NaN of either sign is on top.  HIDDEN: a value for the next layer, the token's scale
// first.  Sum times scale may pass the end of float32 where the value does not (a scale of more than 2^100): there the scale
// goes in 2^24 times smaller, and the fma that adds the bias puts the 2^24 back; both are exact, and the fma costs what the addition does.
// The ReLU is the maximum that keeps a NaN of either sign (infinity and a bias of the other sign make one with the sign bit set here; a maximum
// of bit patterns would take it for a negative value).  Past it the bits order as they are.
// par: the tile's scales and biases in LDS, put there by one load of the wave (read from memory by every lane they would take eight).
__device__ __forceinline__ float int8_mlp_par(const MlpLayer &Y, int ct, int lane) {     // scales in the lower half of the wave, biases in the upper
    return Y.scale[32 * (ct + (lane >> 5) * Y.CT) + (lane & 31)];
}
template <bool HIDDEN>
__device__ __forceinline__ void int8_mlp_values(const i32x16 &acc, const float *par, int h, float s, bool relu, float (&y)[16], unsigned &am) {
    const float floor = HIDDEN || relu ? 0.f : -__builtin_inff();
    const bool far = s > 0x1p100f;                                 // the sums are below 2^24 (at most 1024 channels)
    const float st = far ? s * 0x1p-24f : s, up = far ? 0x1p24f : 1.f;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const f32x4 sc = *reinterpret_cast<const f32x4 *>(par + 8 * g + 4 * h), bi = *reinterpret_cast<const f32x4 *>(par + 32 + 8 * g + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float a = (float)acc[4 * g + j];
            const float v = HIDDEN ? fmaf(a * st * sc[j], up, bi[j]) : a * sc[j] * s + bi[j];
            y[4 * g + j] = int8_max(v, floor);
            if (HIDDEN) am = __float_as_uint(y[4 * g + j]) > am ? __float_as_uint(y[4 * g + j]) : am;
        }
    }
}

// real: channels from the tile's first on; groups of eight past them hold nothing
__device__ __forceinline__ void int8_mlp_top(const float (&e)[16], int real, unsigned &am) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
        if (8 * g < real)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned u = p2n_absbits(e[4 * g + j]);
                am = u > am ? u : am;
            }
}

// codes of an input tile; groups of eight channels past the last one are zero: nothing to form (a level's first layer has six)
__device__ __forceinline__ void int8_mlp_codes(const float (&e)[16], int real, const P2nQ8 &Q, int (&c)[4]) {
    float near = 0.f;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        c[g] = 0;
        if (8 * g < real) c[g] = p2n_q8_four(e + 4 * g, Q, near);
    }
    if (p2n_q8_tie(near, Q)) {
#pragma unroll
        for (int g = 0; g < 4; ++g) c[g] = p2n_q8_decide4(e + 4 * g, Q);
    }
}

// the larger of the two halves of a wave
__device__ __forceinline__ unsigned int8_halves(unsigned am) {
    const auto x = __builtin_amdgcn_permlane32_swap(am, am, false, false);
    return x[0] > x[1] ? x[0] : x[1];
}

// Up to 64 channels everywhere: one wave carries its 32 points through every layer in registers.  Bound by the vector instructions that
// scale the sums and form the next codes, some 12 a value (89 % of the issue slots): 6-32-32-64 with groups of 32 over 16 x 65536 points 47 us,
// of which the memory's share is 7; the maximum by exchanges between lanes instead of in registers: 9 more.
// HT: tiles of 32 channels that the input and the layers between have.  With one, five waves fit a SIMD instead of four (53 -> 47 us).
template <int HT>
__global__ __launch_bounds__(256, HT == 1 ? 5 : 4) void p2n_int8_mlp_narrow_kernel(Int8MlpArgs A) {
    __shared__ __attribute__((aligned(16))) float own[4][HT][64];           // the wave's: parameters of its tiles, in the end scales of its points
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int p = lane & 31, h = lane >> 5;
    const i32x16 zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    const unsigned tile = blockIdx.x * 4 + wave, tiles = (unsigned)A.tiles;          // both below 2^31
    if (tile >= A.total) return;
    const int KT0 = A.layer[0].KT;
    const long b = tile / tiles, l0 = tile % tiles * 32;
    const bool valid = l0 + p < A.L;
    const unsigned off = (unsigned)((4 * h * A.L + (valid ? l0 + p : A.L - 1)) * 4);   // bytes; L <= 2^24 keeps 32 rows below 2^31
    unsigned am = 0;
    float s, v[HT][16];
    int cq[HT][4];
#pragma unroll
    for (int kt = 0; kt < HT; ++kt)
        if (kt < KT0) int8_mlp_load(A.x + b * A.C * A.L, A.L, A.C, kt, off, v[kt]);
#pragma unroll
    for (int kt = 0; kt < HT; ++kt)
        if (kt < KT0) int8_mlp_top(v[kt], A.C - 32 * kt, am);
    s = p2n_q8_scale(int8_halves(am));
    {
        const P2nQ8 Q = p2n_q8_make(s);
#pragma unroll
        for (int kt = 0; kt < HT; ++kt) {
#pragma unroll
            for (int g = 0; g < 4; ++g) cq[kt][g] = 0;
            if (kt < KT0) int8_mlp_codes(v[kt], A.C - 32 * kt, Q, cq[kt]);
        }
    }
#pragma unroll 1
    for (int li = 0; li < A.nl; ++li) {
        const MlpLayer Y = A.layer[li];
        const i32x4 *wf = reinterpret_cast<const i32x4 *>(Y.img) + lane;
        i32x4 x[HT];
#pragma unroll
        for (int kt = 0; kt < HT; ++kt) x[kt] = i32x4{cq[kt][0], cq[kt][1], cq[kt][2], cq[kt][3]};
        // the image has an even number of k-tiles: where the second holds no channels its codes are zero
        if (li == A.nl - 1) {
            if (A.group) {
                own[wave][0][p] = s;
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
#pragma unroll 1
            for (int ct = 0; ct < Y.CT; ++ct) {
                i32x16 acc = zero;
                if (A.group) {
#pragma unroll
                    for (int kt = 0; kt < HT; ++kt) acc = MFMA_I8(x[kt], wf[(ct * Y.KTI + kt) * 64], acc);
                    int8_mlp_groups(A, Y, ct, acc, own[wave][0], b, l0, lane);
                } else {
                    own[wave][0][lane] = int8_mlp_par(Y, ct, lane);
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();
#pragma unroll
                    for (int kt = 0; kt < HT; ++kt) acc = MFMA_I8(wf[(ct * Y.KTI + kt) * 64], x[kt], acc);
                    float y[16];
                    int8_mlp_values<false>(acc, own[wave][0], h, s, A.last_relu, y, am);
                    int8_mlp_out(A, Y.N, b, valid, off, ct, y);
                }
            }
            break;
        }
        float y[HT][16];
        am = 0;
#pragma unroll
        for (int ct = 0; ct < HT; ++ct)
            if (ct < Y.CT) own[wave][ct][lane] = int8_mlp_par(Y, ct, lane);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int ct = 0; ct < HT; ++ct)
            if (ct < Y.CT) {
                i32x16 acc = zero;
#pragma unroll
                for (int kt = 0; kt < HT; ++kt) acc = MFMA_I8(wf[(ct * Y.KTI + kt) * 64], x[kt], acc);
                int8_mlp_values<true>(acc, own[wave][ct], h, s, true, y[ct], am);
            }
        s = p2n_q8_scale(int8_halves(am));
        const P2nQ8 Q = p2n_q8_make(s);
#pragma unroll
        for (int ct = 0; ct < HT; ++ct)
            if (ct < Y.CT) p2n_q8_pack(y[ct], Q, cq[ct]);
    }
}

// Wider layers: NW waves carry 32 points together, a wave its share of the channel tiles.  Codes go round through LDS in operand order; a point's
// maximum is joined over the waves there too.  Two barriers a layer; a layer's first weights are on their way before the last one ends.
// 131-128-128-128-64 over 16 x 8192 points: 41 us (14 vector instructions a value, 63 % of the issue slots, memory 20 us); one wave for all channels: 83.
// IR: k-tiles of the input a wave holds: 4, or 2 where that is enough and five waves a SIMD have work (43 us against 46).  With few
// columns the registers are worth more than the fifth wave (384-256-256 over 515 columns: 9.2 us against 8.6).
template <int NW, bool GROUPS, int IR>
__global__ __launch_bounds__(64 * NW, IR == 2 ? 5 : 4) void p2n_int8_mlp_wide_kernel(Int8MlpArgs A) {
    constexpr int KTI = IR * NW;     // k-tiles of the input, IR a wave; a channel tile a wave: 256 (128) out
    constexpr int AHEAD = 4;                                // weight fragments on their way
    __shared__ __attribute__((aligned(16))) char codes[KTI * 1024];
    __shared__ unsigned top[NW][32];
    __shared__ __attribute__((aligned(16))) float par[NW][64];            // the wave's own row
    __shared__ __attribute__((aligned(16))) float scales[32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int p = lane & 31, h = lane >> 5;
    const unsigned tiles = (unsigned)A.tiles;                    // below 2^31, as the grid
    const long b = blockIdx.x / tiles, l = blockIdx.x % tiles * 32 + p;
    const bool valid = l < A.L;
    const float *xb = A.x + b * A.C * A.L;
    const unsigned off = (unsigned)((4 * h * A.L + (valid ? l : A.L - 1)) * 4);
    const int KT0 = A.layer[0].KT;
    float v[IR][16];
    unsigned am = 0;
#pragma unroll
    for (int i = 0; i < IR; ++i)
        if (wave + NW * i < KT0) int8_mlp_load(xb, A.L, A.C, wave + NW * i, off, v[i]);
    i32x4 w[AHEAD];
    float pw;
    auto ahead = [&](const MlpLayer &Y, int ct) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            w[i] = reinterpret_cast<const i32x4 *>(Y.img)[((ct < Y.CT ? ct : 0) * Y.KTI + (i < Y.KTI ? i : 0)) * 64 + lane];
        pw = int8_mlp_par(Y, ct < Y.CT ? ct : 0, lane);
    };
    ahead(A.layer[0], wave);
#pragma unroll
    for (int i = 0; i < IR; ++i)
        if (wave + NW * i < KT0) int8_mlp_top(v[i], A.C - 32 * (wave + NW * i), am);
    // the largest of every point over the waves -> its scale
    auto join = [&]() __attribute__((always_inline)) {
        const unsigned o = int8_halves(am);
        if (h == 0) top[wave][p] = o;
        __syncthreads();
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < NW; ++i) m = top[i][p] > m ? top[i][p] : m;
        return p2n_q8_scale(m);
    };
    float s = join();
    if (GROUPS && threadIdx.x < 32) scales[p] = s;
    {
        const P2nQ8 Q = p2n_q8_make(s);
#pragma unroll
        for (int i = 0; i < IR; ++i)
            if (wave + NW * i < KT0) {
                int c[4];
                int8_mlp_codes(v[i], A.C - 32 * (wave + NW * i), Q, c);
                *reinterpret_cast<i32x4 *>(codes + ((wave + NW * i) * 64 + lane) * 16) = i32x4{c[0], c[1], c[2], c[3]};
            }
    }
    __syncthreads();
#pragma unroll 1
    for (int li = 0; li < A.nl; ++li) {
        const MlpLayer Y = A.layer[li];
        const bool last = li == A.nl - 1;
        am = 0;
        const bool mine = wave < Y.CT, groups = GROUPS && last;
        if (mine) {
            const i32x4 *wf = reinterpret_cast<const i32x4 *>(Y.img) + (long)wave * Y.KTI * 64 + lane;
            i32x16 acc;
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[e] = 0;
            auto product = [&](auto channels_in_registers) __attribute__((always_inline)) {
                for (int k0 = 0; k0 < Y.KT; k0 += AHEAD) {
#pragma unroll
                    for (int q = 0; q < AHEAD; ++q) {
                        if (k0 + q < Y.KT) {
                            const i32x4 x = *reinterpret_cast<const i32x4 *>(codes + ((k0 + q) * 64 + lane) * 16);
                            acc = channels_in_registers ? MFMA_I8(w[q], x, acc) : MFMA_I8(x, w[q], acc);
                        }
                        if (k0 + q + AHEAD < Y.KT) w[q] = wf[(k0 + q + AHEAD) * 64];
                    }
                }
            };
            if (groups) {
                product(std::false_type{});
                int8_mlp_groups(A, Y, wave, acc, scales, b, l - p, lane);
            } else {
                par[wave][lane] = pw;
                product(std::true_type{});
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                if (last) {
                    int8_mlp_values<false>(acc, par[wave], h, s, A.last_relu, v[0], am);
                    int8_mlp_out(A, Y.N, b, valid, off, wave, v[0]);
                } else {
                    int8_mlp_values<true>(acc, par[wave], h, s, true, v[0], am);
                }
            }
        }
        if (last) break;
        ahead(A.layer[li + 1], wave);
        s = join();                            // behind its barrier every wave has read this layer's codes
        if (GROUPS && threadIdx.x < 32) scales[p] = s;   // read behind the next barrier, by the last layer alone
        if (mine) {
            const P2nQ8 Q = p2n_q8_make(s);
            int c[4];
            p2n_q8_pack(v[0], Q, c);
            *reinterpret_cast<i32x4 *>(codes + (wave * 64 + lane) * 16) = i32x4{c[0], c[1], c[2], c[3]};
        }
        __syncthreads();
    }
}

template <int NW>
static void int8_launch_wide(const Int8MlpArgs &a, int ktm, hipStream_t s) {
    const dim3 grid((unsigned)a.total), blk(64 * NW);
    const bool two = ktm <= 2 * NW && a.total * NW > 4096;          // more waves than four a SIMD hold
    if (two && a.group) hipLaunchKernelGGL((p2n_int8_mlp_wide_kernel<NW, true, 2>), grid, blk, 0, s, a);
    else if (two) hipLaunchKernelGGL((p2n_int8_mlp_wide_kernel<NW, false, 2>), grid, blk, 0, s, a);
    else if (a.group) hipLaunchKernelGGL((p2n_int8_mlp_wide_kernel<NW, true, 4>), grid, blk, 0, s, a);
    else hipLaunchKernelGGL((p2n_int8_mlp_wide_kernel<NW, false, 4>), grid, blk, 0, s, a);
}

// x (B, dims[0], L) -> out (B, dims[nl], L), or (B, dims[nl], L/group) with the maximum over groups of 16 or 32 consecutive
// columns; images_host: HOST array of nl DEVICE pointers (p2n_int8_pack_weight).  ReLU behind every layer but the last,
// behind that one if last_relu.
extern "C" int p2n_int8_mlp(const float *x, int B, long L, int nl, const int *dims, const void *const *images_host, int last_relu, int group,
                            float *out, void *stream_) {
    P2N_REQUIRE(nl >= 1 && nl <= INT8_MAX_LAYERS && dims && images_host, "p2n_int8_mlp: 1..%d layers", INT8_MAX_LAYERS);
    P2N_REQUIRE(B >= 0 && L >= 0 && L <= (1L << 24), "p2n_int8_mlp: bad shape B=%d L=%ld (at most 2^24 columns a cloud)", B, L);
    P2N_REQUIRE(dims[0] >= 1 && dims[0] <= 1024, "p2n_int8_mlp: %d input channels not in [1,1024]", dims[0]);
    for (int l = 1; l <= nl; ++l)
        P2N_REQUIRE(dims[l] >= 1 && dims[l] <= 256, "p2n_int8_mlp: layer %d has %d output channels, not in [1,256]", l - 1, dims[l]);
    P2N_REQUIRE(group == 0 || ((group == 16 || group == 32) && L % group == 0),
                "p2n_int8_mlp: groups of %d columns (0, or 16 or 32 dividing the %ld columns of a cloud)", group, L);
    if (B == 0 || L == 0) return P2N_OK;
    P2N_REQUIRE(x && out, "p2n_int8_mlp: null pointer");
    Int8MlpArgs a = {};
    a.x = x; a.out = out; a.L = L; a.tiles = (L + 31) / 32; a.total = a.tiles * B;
    a.C = dims[0]; a.nl = nl; a.last_relu = last_relu ? 1 : 0; a.group = group;
    int ctm = 0, ktm = (dims[0] + 31) / 32, inside = ktm;      // tiles of the widest layer, of the input; of all that pass from layer to layer
    for (int l = 0; l < nl; ++l) {
        const char *img = (const char *)images_host[l];
        P2N_REQUIRE(img && ((uintptr_t)img & 15) == 0, "p2n_int8_mlp: the image of layer %d is null or not 16-byte aligned", l);
        const Int8Image I = int8_image(dims[l], dims[l + 1]);
        MlpLayer &y = a.layer[l];
        y.img = img; y.scale = (const float *)(img + I.scale); y.bias = (const float *)(img + I.bias);
        y.KT = (dims[l] + 31) / 32; y.KTI = I.KT; y.CT = I.CT; y.N = dims[l + 1];
        if (I.CT > ctm) ctm = I.CT;
        if (l < nl - 1 && I.CT > inside) inside = I.CT;
    }
    const int waves = ctm <= 2 && ktm <= 2 ? 1 : ctm <= 4 && ktm <= 16 ? 4 : 8;     // of 32 columns; a launch holds less than 2^32 threads
    P2N_REQUIRE(a.total * waves * 64 <= (1L << 32) - 512, "p2n_int8_mlp: too many columns (%ld tiles of 32)", a.total);
    hipStream_t s = (hipStream_t)stream_;
    const int ps = p2n_prof_begin(P2N_K_INT8_MLP, s);
    // one wave to 32 points up to 64 channels (fewer registers than four waves would share out), four up to 128, eight up to 256
    if (waves == 1 && inside == 1) hipLaunchKernelGGL(p2n_int8_mlp_narrow_kernel<1>, dim3((unsigned)((a.total + 3) / 4)), dim3(256), 0, s, a);
    else if (waves == 1) hipLaunchKernelGGL(p2n_int8_mlp_narrow_kernel<2>, dim3((unsigned)((a.total + 3) / 4)), dim3(256), 0, s, a);
    else if (waves == 4) int8_launch_wide<4>(a, ktm, s);
    else int8_launch_wide<8>(a, ktm, s);
    p2n_prof_end(ps, s);
    P2N_CHECK_HIP(hipGetLastError());
    return P2N_OK;
}

// ---------------------------------------------------------------- maximum of consecutive values, NaN kept
__global__ __launch_bounds__(256) void p2n_int8_rowmax_kernel(const float *__restrict__ in, long rows, int ns, float *__restrict__ out) {
    const long r = (long)blockIdx.x * 256 + threadIdx.x;
    if (r >= rows) return;
    int m = int8_key(in[r * ns]);
    for (int i = 1; i < ns; ++i) {
        const int k = int8_key(in[r * ns + i]);
        m = k > m ? k : m;
    }
    out[r] = __int_as_float(int8_unkey(m));
}

extern "C" int p2n_max_of_columns(const float *in, long rows, int ns, float *out, void *stream_) {
    P2N_REQUIRE(rows >= 0 && ns >= 1 && rows <= (1L << 32) - 256, "p2n_max_of_columns: bad shape");
    if (rows == 0) return P2N_OK;
    P2N_REQUIRE(in && out, "p2n_max_of_columns: null pointer");
    hipLaunchKernelGGL(p2n_int8_rowmax_kernel, dim3((unsigned)((rows + 255) / 256)), dim3(256), 0, (hipStream_t)stream_, in, rows, ns, out);
    P2N_CHECK_HIP(hipGetLastError());
    return P2N_OK;
}
