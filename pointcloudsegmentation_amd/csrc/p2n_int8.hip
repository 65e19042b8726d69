// Products in 8-bit integers for gfx950 (MI355X), one scale for a token (a point) and one for an output channel:
//     (sx_t, qx_t) = 8-bit rule over the K values of token t        (sw_n, qw_n) = 8-bit rule over row n of W (N, K)
//     y[t][n] = fl(fl(fl(sum_k qx qw) * sw_n) * sx_t) + b_n, then ReLU if asked
// The sum is exact in int32 (K <= 65536 keeps it below 2^31); its conversion to float32 and the two products round once
// each.  The reference has no 8-bit path (its layers are Conv1d, reference point2net.py:9-34): the formulas above are the
// specification.  Two operators share the weight image and the rule (p2n_q8.h):
//   p2n_int8_linear  rows of K values (tokens), float32 or bfloat16
//   p2n_int8_mlp     the layers of a shared MLP over the columns of (B, C, L), register-resident
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

// one wave per channel: maximum, scale, codes
__global__ __launch_bounds__(256) void p2n_int8_pack_kernel(const float *__restrict__ W, const float *__restrict__ bias, int K, int N,
                                                            int CT, int KT, char *__restrict__ img, float *__restrict__ scale,
                                                            float *__restrict__ bimg) {
    const int lane = threadIdx.x & 63;
    const int n = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (n >= 32 * CT) return;
    const float *w = W + (long)n * K;
    unsigned am = 0;
    if (n < N)
        for (int k = lane; k < K; k += 64) {
            const unsigned b = p2n_absbits(w[k]);
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
        bimg[n] = n < N && bias ? bias[n] : 0.f;
    }
    const int ct = n >> 5, r = n & 31;
    const bool bad = !(s == s);
    for (int k4 = lane; k4 < 8 * KT; k4 += 64) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = 4 * k4 + j;
            v[j] = (n < N && k < K) ? w[k] : 0.f;
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

extern "C" int p2n_int8_pack_weight(const float *W, const float *bias, int K, int N, void *image, void *stream_) {
    P2N_REQUIRE(K >= 1 && K <= INT8_MAX_K && N >= 1 && N <= INT8_MAX_N, "p2n_int8_pack_weight: K=%d or N=%d not in [1,%d]", K, N, INT8_MAX_K);
    P2N_REQUIRE(W && image, "p2n_int8_pack_weight: null pointer");
    P2N_REQUIRE(((uintptr_t)image & 15) == 0, "p2n_int8_pack_weight: the image must be 16-byte aligned");
    const Int8Image I = int8_image(K, N);
    char *img = (char *)image;
    hipStream_t s = (hipStream_t)stream_;
    const int ps = p2n_prof_begin(P2N_K_INT8_PACK, s);
    hipLaunchKernelGGL(p2n_int8_pack_kernel, dim3(8 * I.CT), dim3(256), 0, s, W, bias, K, N, I.CT, I.KT, img, (float *)(img + I.scale),
                       (float *)(img + I.bias));
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

// The same into fragments: tile tt of 32 tokens, fragment tt * KT + kt laid out as in the weight image; scales (32 TT).
// A workgroup takes one tile of tokens; lane = (token, half), a wave every fourth k-tile.  Tokens behind the last one
// have code and scale 0.
template <typename TX>
__global__ __launch_bounds__(256) void p2n_int8_tile_kernel(const TX *__restrict__ x, long T, int K, long ld, int KT, char *__restrict__ img,
                                                            float *__restrict__ scale) {
    __shared__ unsigned sh[4][32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int r = lane & 31, h = lane >> 5;
    const long tt = blockIdx.x, t = tt * 32 + r;
    const TX *row = x + (t < T ? t : T - 1) * ld;
    unsigned am = 0;
    for (int kt = wave; kt < KT; kt += 4)
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = 32 * kt + 8 * g + 4 * h + j;
                const unsigned b = p2n_absbits(int8_load(row + (k < K ? k : K - 1)));   // a value read twice moves no maximum
                am = b > am ? b : am;
            }
    {
        const unsigned o = (unsigned)__shfl_xor((int)am, 32);
        am = o > am ? o : am;
    }
    if (h == 0) sh[wave][r] = am;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) am = sh[w][r] > am ? sh[w][r] : am;
    const float s = t < T ? p2n_q8_scale(am) : 0.f;
    const P2nQ8 Q = p2n_q8_make(s);
    if (wave == 0 && h == 0) scale[t] = s;
    for (int kt = wave; kt < KT; kt += 4) {
        float v[16];
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = 32 * kt + 8 * g + 4 * h + j;
                const float e = int8_load(row + (k < K ? k : K - 1));
                v[4 * g + j] = k < K ? e : 0.f;
            }
        int c[4];
        p2n_q8_pack(v, Q, c);
        *reinterpret_cast<i32x4 *>(img + ((tt * KT + kt) * 64 + lane) * 16) = i32x4{c[0], c[1], c[2], c[3]};
    }
}

__device__ __forceinline__ void int8_store(float *p, float v) { *p = v; }
__device__ __forceinline__ void int8_store(__bf16 *p, float v) { *p = (__bf16)v; }

__device__ __forceinline__ float int8_value(int acc, float sx, float sw, float b, int relu) {
    const float v = (float)acc * sw * sx + b;   // the token's scale last: it may be as large as float32 goes
    return relu && v <= 0.f ? 0.f : v;   // a NaN stays
}

// ---------------------------------------------------------------- product of fragments
// D = X . W^T, registers = tokens, lane = channel: a workgroup of four waves makes 128 tokens x 128 channels, a wave 64 x 64.
template <typename TY>
__global__ __launch_bounds__(256) void p2n_int8_gemm_kernel(const char *__restrict__ xi, const float *__restrict__ sx, const char *__restrict__ wi,
                                                            const float *__restrict__ sw, const float *__restrict__ bias, long T, int N, int TT, int CT,
                                                            int KT, int relu, TY *__restrict__ y) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int r = lane & 31, h = lane >> 5;
    const int t0 = blockIdx.y * 4 + (wave >> 1) * 2, c0 = blockIdx.x * 4 + (wave & 1) * 2;
    if (t0 >= TT || c0 >= CT) return;
    const i32x4 *xa = reinterpret_cast<const i32x4 *>(xi) + lane, *wb = reinterpret_cast<const i32x4 *>(wi) + lane;
    const int t1 = t0 + 1 < TT ? t0 + 1 : t0, c1 = c0 + 1 < CT ? c0 + 1 : c0;
    i32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][c][e] = 0;
    for (int kt = 0; kt < KT; ++kt) {
        const i32x4 a0 = xa[((long)t0 * KT + kt) * 64], a1 = xa[((long)t1 * KT + kt) * 64];
        const i32x4 b0 = wb[((long)c0 * KT + kt) * 64], b1 = wb[((long)c1 * KT + kt) * 64];
        acc[0][0] = MFMA_I8(a0, b0, acc[0][0]);
        acc[0][1] = MFMA_I8(a0, b1, acc[0][1]);
        acc[1][0] = MFMA_I8(a1, b0, acc[1][0]);
        acc[1][1] = MFMA_I8(a1, b1, acc[1][1]);
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int n = 32 * (c0 + c) + r;
        if (n >= N) continue;
        const float w = sw[n], b = bias[n];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const long t = 32L * (t0 + i) + 8 * (e >> 2) + 4 * h + (e & 3);
                if (t < T) int8_store(y + t * N + n, int8_value(acc[i][c][e], sx[t], w, b, relu));
            }
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
    const dim3 grid((unsigned)((T + 3) / 4)), blk(256);
    const int ps = p2n_prof_begin(P2N_K_INT8_TOKENS, s);
    if (bf16) hipLaunchKernelGGL(p2n_quantize_tokens_kernel<__bf16>, grid, blk, 0, s, (const __bf16 *)x, T, K, ld, codes, scale);
    else hipLaunchKernelGGL(p2n_quantize_tokens_kernel<float>, grid, blk, 0, s, (const float *)x, T, K, ld, codes, scale);
    p2n_prof_end(ps, s);
    P2N_CHECK_HIP(hipGetLastError());
    return P2N_OK;
}

extern "C" size_t p2n_int8_linear_workspace_bytes(long T, int K, int N) {
    if (T < 1 || T >= (1L << 31) || K < 1 || K > INT8_MAX_K || N < 1 || N > INT8_MAX_N) return 0;
    return int8_tiles_bytes(T, K);
}

template <typename TX>
static int int8_linear_run(const TX *x, long T, int K, long ld, const char *img, int N, int relu, TX *y, char *ws, hipStream_t s) {
    const Int8Image I = int8_image(K, N);
    const long TT = (T + 31) / 32;
    float *sx = (float *)(ws + (size_t)TT * I.KT * 1024);
    hipLaunchKernelGGL(p2n_int8_tile_kernel<TX>, dim3((unsigned)TT), dim3(256), 0, s, x, T, K, ld, I.KT, ws, sx);
    P2N_CHECK_HIP(hipGetLastError());
    for (long t0 = 0; t0 < TT; t0 += 4L * 65535) {   // grid.y holds 65,535 workgroups
        const long n = TT - t0 < 4L * 65535 ? TT - t0 : 4L * 65535;
        const long rows = T - 32 * t0;
        hipLaunchKernelGGL(p2n_int8_gemm_kernel<TX>, dim3((unsigned)((I.CT + 3) / 4), (unsigned)((n + 3) / 4)), dim3(256), 0, s, ws + (size_t)t0 * I.KT * 1024,
                           sx + 32 * t0, img, (const float *)(img + I.scale), (const float *)(img + I.bias), rows, N, (int)n, I.CT, I.KT, relu,
                           y + 32 * t0 * N);
        P2N_CHECK_HIP(hipGetLastError());
    }
    return P2N_OK;
}

extern "C" int p2n_int8_linear(const void *x, int bf16, long T, int K, long ld, const void *image, int N, int relu, void *y, void *workspace,
                               size_t workspace_bytes, void *stream_) {
    P2N_REQUIRE(T >= 0 && T < (1L << 31) && K >= 1 && K <= INT8_MAX_K && N >= 1 && N <= INT8_MAX_N && ld >= K,
                "p2n_int8_linear: bad shape T=%ld K=%d N=%d ld=%ld", T, K, N, ld);
    if (T == 0) return P2N_OK;
    P2N_REQUIRE(x && image && y, "p2n_int8_linear: null pointer");
    const size_t need = p2n_int8_linear_workspace_bytes(T, K, N);
    if (!workspace || workspace_bytes < need) {
        p2n_set_error("p2n_int8_linear: workspace %zu bytes < required %zu", workspace_bytes, need);
        return P2N_EWORKSPACE;
    }
    P2N_REQUIRE((((uintptr_t)workspace | (uintptr_t)image) & 15) == 0, "p2n_int8_linear: workspace and image must be 16-byte aligned");
    hipStream_t s = (hipStream_t)stream_;
    const int ps = p2n_prof_begin(P2N_K_INT8_GEMM, s);
    const int rc = bf16 ? int8_linear_run<__bf16>((const __bf16 *)x, T, K, ld, (const char *)image, N, relu, (__bf16 *)y, (char *)workspace, s)
                        : int8_linear_run<float>((const float *)x, T, K, ld, (const char *)image, N, relu, (float *)y, (char *)workspace, s);
    p2n_prof_end(ps, s);
    return rc;
}

// ---------------------------------------------------------------- shared MLP, register-resident
// Lane = point, registers = channels (D = W . X): a wave carries 32 points through every layer.  The 32 x 32 product leaves
// channel 32ct + 8g + 4h + j of a lane's point in register 4g + j of its half h; four neighbours packed to a dword are the
// operand of the next layer in the k order of the weight image.  Nothing of a hidden layer leaves the wave: its scale is a
// maximum over the lane's registers and the other half (one shuffle).
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

// The 16 channels 32kt + 8g + 4h + j of this lane's point.  The resource starts at row 32kt and ends with the cloud's last
// row, so channels past C read as zero; `off` is the lane's byte offset (half's rows and column).
__device__ __forceinline__ void int8_mlp_load(const float *xb, long L, int C, int kt, int off, float (&v)[16]) {
    const long left = (long)(C - 32 * kt) * L * 4;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(xb + 32L * kt * L), 0,
                                                                         (int)(left < 0xFFFFFFFFL ? left : 0xFFFFFFFFL), 0x00020000);
#pragma unroll
    for (int e = 0; e < 16; ++e)
        v[e] = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, off + (int)((8 * (e >> 2) + (e & 3)) * L * 4), 0, 0));
}

// CTM: channel tiles of the widest layer; KTM >= CTM: k-tiles of the widest operand
template <int CTM, int KTM>
__global__ __launch_bounds__(256, CTM <= 2 ? 4 : CTM <= 4 ? 3 : KTM <= 8 ? 2 : 1) void p2n_int8_mlp_kernel(Int8MlpArgs A) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int p = lane & 31, h = lane >> 5;
    for (long tile = (long)blockIdx.x * 4 + wave; tile < A.total; tile += (long)gridDim.x * 4) {
        const long b = tile / A.tiles, l = (tile % A.tiles) * 32 + p;
        const bool valid = l < A.L;
        const float *xb = A.x + b * A.C * A.L;
        const int off = (int)((4 * h * A.L + (valid ? l : A.L - 1)) * 4);   // bytes; L <= 2^24 keeps 32 rows below 2^31
        const int KT0 = A.layer[0].KT;
        unsigned am = 0;
#pragma unroll 1
        for (int kt = 0; kt < KT0; ++kt) {
            float v[16];
            int8_mlp_load(xb, A.L, A.C, kt, off, v);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const unsigned u = p2n_absbits(v[e]);
                am = u > am ? u : am;
            }
        }
        unsigned o = (unsigned)__shfl_xor((int)am, 32);
        float s = p2n_q8_scale(o > am ? o : am);
        int cq[KTM][4];
        {
            const P2nQ8 Q = p2n_q8_make(s);
#pragma unroll
            for (int kt = 0; kt < KTM; ++kt)
                if (kt < KT0) {
                    float v[16];
                    int8_mlp_load(xb, A.L, A.C, kt, off, v);
                    p2n_q8_pack(v, Q, cq[kt]);
                    __builtin_amdgcn_sched_barrier(0);   // one tile at a time: interleaved tiles cost registers
                }
        }
#pragma unroll 1
        for (int li = 0; li < A.nl; ++li) {
            const MlpLayer Y = A.layer[li];
            const bool last = li == A.nl - 1;
            const bool relu = !last || A.last_relu;
            const i32x4 *wf = reinterpret_cast<const i32x4 *>(Y.img) + lane;
            float y[CTM][16];
            am = 0;
#pragma unroll
            for (int ct = 0; ct < CTM; ++ct)
                if (ct < Y.CT) {
                    i32x16 acc;
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[e] = 0;
#pragma unroll
                    for (int kt = 0; kt < KTM; ++kt)
                        if (kt < Y.KT) acc = MFMA_I8(wf[(ct * Y.KTI + kt) * 64], (i32x4{cq[kt][0], cq[kt][1], cq[kt][2], cq[kt][3]}), acc);
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x4 sc = *reinterpret_cast<const f32x4 *>(Y.scale + 32 * ct + 8 * g + 4 * h);
                        const f32x4 bi = *reinterpret_cast<const f32x4 *>(Y.bias + 32 * ct + 8 * g + 4 * h);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            float v = (float)acc[4 * g + j] * sc[j] * s + bi[j];
                            if (relu) v = v <= 0.f ? 0.f : v;   // a NaN stays
                            y[ct][4 * g + j] = v;
                            const unsigned u = p2n_absbits(v);
                            am = u > am ? u : am;
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            if (last) {
                const long W = A.group ? A.L / A.group : A.L;   // columns of a result row
                float *ob = A.out + b * Y.N * W;
#pragma unroll
                for (int ct = 0; ct < CTM; ++ct)
                    if (ct < Y.CT) {
                        // the resource starts at row 32ct and ends with the cloud's last row: channels past N are not written
                        const long left = (long)(Y.N - 32 * ct) * W * 4;
                        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                            ob + 32L * ct * W, 0, (int)(left < 0xFFFFFFFFL ? left : 0xFFFFFFFFL), 0x00020000);
                        if (!A.group) {
                            if (valid) {
#pragma unroll
                                for (int e = 0; e < 16; ++e)
                                    __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(y[ct][e]), rs, off + (int)((8 * (e >> 2) + (e & 3)) * W * 4), 0, 0);
                            }
                        } else {
                            // maximum over 32 (or 16) neighbouring points of every channel: the registers shrink 16 -> 1 while
                            // the lanes of a 16-lane row pair up; lane i of a row ends with register i's channel
                            int m[16];
#pragma unroll
                            for (int e = 0; e < 16; ++e) m[e] = int8_key(y[ct][e]);
                            p2n_halve_max<8, 0xB1>(m, lane & 1);
                            p2n_halve_max<4, 0x4E>(m, lane & 2);
                            p2n_halve_max<2, 0x124>(m, lane & 4);
                            p2n_halve_max<1, 0x128>(m, lane & 8);
                            if (A.group == 32) {
                                const int t = __builtin_amdgcn_ds_swizzle(m[0], 0x401F);   // lane ^ 16
                                m[0] = t > m[0] ? t : m[0];
                            }
                            const int i = lane & 15, c = 8 * (i >> 2) + 4 * h + (i & 3);
                            const int q = A.group == 32 ? (int)(l >> 5) : (int)(l >> 4);
                            if (valid && (A.group == 16 || !(lane & 16)))
                                __builtin_amdgcn_raw_buffer_store_b32(int8_unkey(m[0]), rs, (int)((c * W + q) * 4), 0, 0);
                        }
                    }
                break;
            }
            o = (unsigned)__shfl_xor((int)am, 32);
            s = p2n_q8_scale(o > am ? o : am);
            const P2nQ8 Q = p2n_q8_make(s);
#pragma unroll
            for (int ct = 0; ct < CTM; ++ct)
                if (ct < Y.CT) {
                    p2n_q8_pack(y[ct], Q, cq[ct]);
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
    }
}

template <int CTM, int KTM>
static void launch_int8_mlp(const Int8MlpArgs &a, hipStream_t s) {
    const long wgs = (a.total + 3) / 4;
    hipLaunchKernelGGL((p2n_int8_mlp_kernel<CTM, KTM>), dim3((unsigned)(wgs < 65536 ? wgs : 65536)), dim3(256), 0, s, a);
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
    int ctm = 0, ktm = (dims[0] + 31) / 32;
    for (int l = 0; l < nl; ++l) {
        const char *img = (const char *)images_host[l];
        P2N_REQUIRE(img && ((uintptr_t)img & 15) == 0, "p2n_int8_mlp: the image of layer %d is null or not 16-byte aligned", l);
        const Int8Image I = int8_image(dims[l], dims[l + 1]);
        MlpLayer &y = a.layer[l];
        y.img = img; y.scale = (const float *)(img + I.scale); y.bias = (const float *)(img + I.bias);
        y.KT = (dims[l] + 31) / 32; y.KTI = I.KT; y.CT = I.CT; y.N = dims[l + 1];
        if (I.CT > ctm) ctm = I.CT;
    }
    if (ctm > ktm) ktm = ctm;
    hipStream_t s = (hipStream_t)stream_;
    const int ps = p2n_prof_begin(P2N_K_INT8_MLP, s);
    if (ktm > 8) {
        if (ktm > 16) launch_int8_mlp<8, 32>(a, s);
        else launch_int8_mlp<8, 16>(a, s);
    } else if (ctm > 4) {
        launch_int8_mlp<8, 8>(a, s);
    } else if (ctm > 2) {
        if (ktm > 4) launch_int8_mlp<4, 8>(a, s);
        else launch_int8_mlp<4, 4>(a, s);
    } else {
        if (ktm > 2) launch_int8_mlp<2, 8>(a, s);
        else launch_int8_mlp<2, 2>(a, s);
    }
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
    P2N_REQUIRE(rows >= 0 && ns >= 1 && rows < (1L << 38), "p2n_max_of_columns: bad shape");
    if (rows == 0) return P2N_OK;
    P2N_REQUIRE(in && out, "p2n_max_of_columns: null pointer");
    hipLaunchKernelGGL(p2n_int8_rowmax_kernel, dim3((unsigned)((rows + 255) / 256)), dim3(256), 0, (hipStream_t)stream_, in, rows, ns, out);
    P2N_CHECK_HIP(hipGetLastError());
    return P2N_OK;
}
