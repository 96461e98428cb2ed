// Products of 8-bit rows with a scale for each token and each channel, and the fold that ends a transposed convolution made
// as such a product: what draws alignments from a trained generator (the reference's ConvTranspose2d stacks,
// src/layers.py:91-147, in evaluation).
//
//   s_t = max_k |x_tk| / 127        q_tk = rint(x_tk 127 / max_k |x_tk|)        (tokens here, channels once beforehand)
//   y_tn = s_t s_n sum_k q_tk w_nk + bias_n
//
// The sum is exact: whole numbers in 32 bits (K <= 131072 keeps 127^2 K below 2^31).  A row's largest magnitude counts as at
// least 2^-100, which keeps both quotients finite; a row that holds an infinity or a NaN gets codes 0 and the scale NaN, so
// that its whole row of y is NaN and no other row is touched.
#include "../../include/pgan_hip.h"
#include "pgan_common.h"

// each product and sum rounded by itself: codes are the same wherever the formulas are evaluated in fp32
#pragma clang fp contract(off)

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

template <int TYPE>
struct Elem {
    using type = float;
};
template <>
struct Elem<1> {
    using type = uint16_t;
};
template <>
struct Elem<2> {
    using type = _Float16;
};
template <int TYPE>
__device__ __forceinline__ float to_f32(typename Elem<TYPE>::type x) {
    if constexpr (TYPE == 1) return __builtin_bit_cast(float, (uint32_t)x << 16);
    else return (float)x;
}
template <int TYPE>
__device__ __forceinline__ typename Elem<TYPE>::type from_f32(float x) {
    if constexpr (TYPE == 1) {      // to the nearest, ties to even
        const uint32_t u = __builtin_bit_cast(uint32_t, x);
        return x != x ? (uint16_t)((u >> 16) | 0x40u) : (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
    } else {
        return (typename Elem<TYPE>::type)x;
    }
}

// magnitude as a pattern: ordered like the magnitudes, infinities above every number and NaN above those
__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }
// maximum over groups of G lanes (a power of two), in every lane of the group
template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
    for (int d = 1; d < G; d <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d, 64));
    return v;
}
struct RowScale {
    float inv, scale;       // x inv: code; code scale: value
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return RowScale{0.f, __builtin_nanf("")};
    const float amax = __builtin_fmaxf(__builtin_bit_cast(float, amax_bits), 0x1p-100f);
    return RowScale{127.f / amax, amax * (float)(1.0 / 127)};
}
// the code of x; a row without a finite maximum (inv = 0) has none but 0
__device__ __forceinline__ int code_of(float x, float inv) { return inv == 0.f ? 0 : (int)rintf(x * inv); }
__device__ __forceinline__ float slope(float x, bool lrelu) { return lrelu && !(x > 0.f) ? x * PGAN_SLOPE : x; }

// ---- rows to codes ------------------------------------------------------------------------------------------------
// one row a wave
template <int TYPE>
__global__ __launch_bounds__(256) void quant_rows_kernel(const typename Elem<TYPE>::type* __restrict__ x, long long ldx,
                                                         int8_t* __restrict__ q, long long ldq, float* __restrict__ scale,
                                                         long long rows, int K, int lrelu) {
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= rows) return;
    const typename Elem<TYPE>::type* xr = x + row * ldx;
    uint32_t mx = 0;
    for (int k = lane; k < K; k += 64) mx = max(mx, magnitude(slope(to_f32<TYPE>(xr[k]), lrelu)));
    const RowScale rs = row_scale(group_max<64>(mx));
    int8_t* qr = q + row * ldq;
    for (int k = lane; k < K; k += 64) qr[k] = (int8_t)code_of(slope(to_f32<TYPE>(xr[k]), lrelu), rs.inv);
    if (lane == 0) scale[row] = rs.scale;
}

// ---- the product --------------------------------------------------------------------------------------------------
// A block of four waves makes 128 tokens x 128 channels, a wave 64 x 64 as 2 x 2 tiles of 32 x 32 (i32 <- i8, 32 deep).
// Stages of 128 bytes along K go through registers into LDS, where chunk c (16 bytes) of row r lies at slot r ^ 2c of its
// 32 rows: a stage's global reads are whole 128-byte lines and neither side of LDS has bank conflicts.
constexpr int GT = 128, GN = 128, GK = 128;

__device__ __forceinline__ int lds_slot(int row, int c) { return (row >> 5) * (32 * GK / 16) + c * 32 + ((row & 31) ^ (2 * c)); }

// 16 bytes of a row from byte k on, zero from byte K on (rows are readable up to the next multiple of 16)
__device__ __forceinline__ i32x4 load16(const int8_t* row, int k, int K) {
    i32x4 v = {0, 0, 0, 0};
    if (k < K) {
        v = *reinterpret_cast<const i32x4*>(row + k);
        if (k + 16 > K) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int left = K - k - 4 * e;
                v[e] = left >= 4 ? v[e] : left <= 0 ? 0 : v[e] & ((1 << (8 * left)) - 1);
            }
        }
    }
    return v;
}

template <int TYPE>
__global__ __launch_bounds__(256) void gemm_q8_kernel(const int8_t* __restrict__ q, long long ldq, const float* __restrict__ qs,
                                                      const int8_t* __restrict__ w, long long ldw,
                                                      const float* __restrict__ ws, const float* __restrict__ bias,
                                                      typename Elem<TYPE>::type* __restrict__ y, long long ldy, long long T,
                                                      int N, int K) {
    __shared__ i32x4 sx[GT * GK / 16], sw[GN * GK / 16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long long t0 = (long long)blockIdx.y * GT;
    const int n0 = blockIdx.x * GN;
    i32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
    const int c = tid & 7;
    for (int k0 = 0; k0 < K; k0 += GK) {
        i32x4 vx[4], vw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {       // rows past the end repeat the last one; what they give is not stored
            const int r = (tid >> 3) + 32 * i;
            const long long t = t0 + r < T ? t0 + r : T - 1;
            const int n = n0 + r < N ? n0 + r : N - 1;
            vx[i] = load16(q + t * ldq, k0 + 16 * c, K);
            vw[i] = load16(w + (long long)n * ldw, k0 + 16 * c, K);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = (tid >> 3) + 32 * i;
            sx[lds_slot(r, c)] = vx[i];
            sw[lds_slot(r, c)] = vw[i];
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < GK / 32; ++s) {
            const int cc = 2 * s + (lane >> 5);
            i32x4 a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[i] = sw[lds_slot((wave & 1) * 64 + 32 * i + (lane & 31), cc)];
                b[i] = sx[lds_slot((wave >> 1) * 64 + 32 * i + (lane & 31), cc)];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[i], b[j], acc[i][j], 0, 0, 0);
        }
    }
    // channel (within 32): e % 4 + 8 (e / 4) + 4 (lane / 32); token: lane % 32
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const long long t = t0 + (wave >> 1) * 64 + 32 * j + (lane & 31);
        if (t >= T) continue;
        const float st = qs[t];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int n = n0 + (wave & 1) * 64 + 32 * i + (e & 3) + 8 * (e >> 2) + 4 * (lane >> 5);
                if (n >= N) continue;
                float v = (float)acc[i][j][e] * (st * ws[n]);
                if (bias) v = v + bias[n];
                y[t * ldy + n] = from_f32<TYPE>(v);
            }
    }
}

// ---- the fold -----------------------------------------------------------------------------------------------------
// y: one row of 4 x 4 taps x C channels for each of B x H x W pixels; output pixel (oh, ow) of 2H x 2W is the sum of the
// (up to) four taps (kh, kw) of pixels (ih, iw) with oh = 2 ih + kh - 1, ow = 2 iw + kw - 1.  An even row takes tap 1 of
// its own input row and tap 3 of the one before, an odd row tap 2 of its own and tap 0 of the one after; so do columns.
struct Taps {
    long long at[2][2];     // first element of the tap's channels, -1: outside
};
__device__ __forceinline__ Taps taps_of(long long pix, int H, int W, int C) {
    const int W2 = 2 * W, H2 = 2 * H;
    const int ow = (int)(pix % W2), oh = (int)(pix / W2 % H2);
    const long long b = pix / W2 / H2;
    const int ih = oh >> 1, iw = ow >> 1;
    const int h2 = oh & 1 ? ih + 1 : ih - 1, w2 = ow & 1 ? iw + 1 : iw - 1;
    const int ka = oh & 1 ? 2 : 1, kb = oh & 1 ? 0 : 3, la = ow & 1 ? 2 : 1, lb = ow & 1 ? 0 : 3;
    const bool hok = h2 >= 0 && h2 < H, wok = w2 >= 0 && w2 < W;
    const long long ra = (b * H + ih) * W, rb = (b * H + h2) * W;
    Taps t;
    t.at[0][0] = ((ra + iw) * 16 + ka * 4 + la) * C;
    t.at[1][0] = hok ? ((rb + iw) * 16 + kb * 4 + la) * C : -1;
    t.at[0][1] = wok ? ((ra + w2) * 16 + ka * 4 + lb) * C : -1;
    t.at[1][1] = hok && wok ? ((rb + w2) * 16 + kb * 4 + lb) * C : -1;
    return t;
}
template <int TYPE>
__device__ __forceinline__ float folded(const typename Elem<TYPE>::type* y, const Taps& t, int c, const float* shift) {
    const auto get = [&](int i, int j) { return t.at[i][j] < 0 ? 0.f : to_f32<TYPE>(y[t.at[i][j] + c]); };
    const float o = (get(0, 0) + get(1, 0)) + (get(0, 1) + get(1, 1));
    return shift ? o + shift[c] : o;
}

// one output pixel a wave: sum, LeakyReLU, codes
template <int TYPE>
__global__ __launch_bounds__(256) void up_fold_q8_kernel(const typename Elem<TYPE>::type* __restrict__ y,
                                                         const float* __restrict__ shift, int8_t* __restrict__ q,
                                                         long long ldq, float* __restrict__ scale, long long pixels, int H,
                                                         int W, int C) {
    const long long pix = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (pix >= pixels) return;
    const Taps t = taps_of(pix, H, W, C);
    uint32_t mx = 0;
    for (int c = lane; c < C; c += 64) mx = max(mx, magnitude(slope(folded<TYPE>(y, t, c, shift), true)));
    const RowScale rs = row_scale(group_max<64>(mx));
    for (int c = lane; c < C; c += 64) q[pix * ldq + c] = (int8_t)code_of(slope(folded<TYPE>(y, t, c, shift), true), rs.inv);
    if (lane == 0) scale[pix] = rs.scale;
}

template <int TYPE>
__global__ __launch_bounds__(256) void up_fold_kernel(const typename Elem<TYPE>::type* __restrict__ y,
                                                      const float* __restrict__ shift, float* __restrict__ out,
                                                      long long pixels, int H, int W, int C, int act) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= pixels * C) return;
    const long long pix = i / C;
    float o = folded<TYPE>(y, taps_of(pix, H, W, C), (int)(i % C), shift);
    if (act == 1) o = 1.f / (1.f + expf(-o));
    if (act == 2) o = tanhf(o);
    out[i] = o;
}

// threads of one launch stay below 2^32
constexpr long long MAX_BLOCKS = 0xffffff;
inline bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
inline int type_bytes(int type) { return type == 0 ? 4 : 2; }

template <class F>
inline int by_type(int type, F f) {
    switch (type) {
        case 0: f(std::integral_constant<int, 0>{}); break;
        case 1: f(std::integral_constant<int, 1>{}); break;
        default: f(std::integral_constant<int, 2>{}); break;
    }
    return pgan_launch_status();
}

}  // namespace

extern "C" {

int pgan_quant_rows(const void* x, int x_type, long long ldx, void* q, long long ldq, float* scale, long long rows, int K,
                    int lrelu, hipStream_t st) {
    if (rows < 0 || K < 1 || x_type < 0 || x_type > 2) return PGAN_EINVAL;
    if (rows == 0) return PGAN_OK;
    if (!x || !q || !scale || !aligned(x, type_bytes(x_type)) || !aligned(scale, 4) || ldx < K || ldq < K) return PGAN_EINVAL;
    const long long blocks = (rows + 3) / 4;
    if (blocks > MAX_BLOCKS) return PGAN_EINVAL;
    return by_type(x_type, [&](auto t) {
        quant_rows_kernel<t.value><<<(unsigned)blocks, 256, 0, st>>>(static_cast<const typename Elem<t.value>::type*>(x), ldx,
                                                                      static_cast<int8_t*>(q), ldq, scale, rows, K, lrelu);
    });
}

int pgan_gemm_q8(const void* q, long long ldq, const float* q_scale, const void* w, long long ldw, const float* w_scale,
                 const float* bias, void* y, int y_type, long long ldy, long long T, int N, int K, hipStream_t st) {
    if (T < 0 || N < 1 || K < 1 || K > 131072 || y_type < 0 || y_type > 2) return PGAN_EINVAL;
    if (T == 0) return PGAN_OK;
    if (!q || !q_scale || !w || !w_scale || !y || !aligned(q, 16) || !aligned(w, 16) || ldq % 16 || ldw % 16 || ldq < K
        || ldw < K || ldy < N || !aligned(y, type_bytes(y_type)))
        return PGAN_EINVAL;
    const long long bt = (T + GT - 1) / GT;
    const int bn = (N + GN - 1) / GN;
    if (bt > 65535) return PGAN_EINVAL;
    return by_type(y_type, [&](auto t) {
        gemm_q8_kernel<t.value><<<dim3((unsigned)bn, (unsigned)bt), 256, 0, st>>>(
            static_cast<const int8_t*>(q), ldq, q_scale, static_cast<const int8_t*>(w), ldw, w_scale, bias,
            static_cast<typename Elem<t.value>::type*>(y), ldy, T, N, K);
    });
}

int pgan_linear_q8(const void* x, int x_type, long long ldx, void* q, long long ldq, float* q_scale, const void* w,
                   long long ldw, const float* w_scale, const float* bias, void* y, int y_type, long long ldy, long long T,
                   int N, int K, int lrelu, hipStream_t st) {
    if (T < 0 || N < 1 || K < 1 || K > 131072 || x_type < 0 || x_type > 2 || y_type < 0 || y_type > 2) return PGAN_EINVAL;
    if (T == 0) return PGAN_OK;
    if (!x || !w || !w_scale || !y || !q || !q_scale || !aligned(q, 16) || !aligned(w, 16) || ldq % 16 || ldw % 16
        || ldq < K || ldw < K || ldx < K || ldy < N || !aligned(x, type_bytes(x_type)) || !aligned(y, type_bytes(y_type)))
        return PGAN_EINVAL;
    const int rc = pgan_quant_rows(x, x_type, ldx, q, ldq, q_scale, T, K, lrelu, st);
    return rc ? rc : pgan_gemm_q8(q, ldq, q_scale, w, ldw, w_scale, bias, y, y_type, ldy, T, N, K, st);
}

int pgan_up_fold_q8(const void* y, int y_type, const float* shift, void* q, long long ldq, float* scale, int B, int H, int W,
                    int C, hipStream_t st) {
    if (B < 0 || H < 1 || W < 1 || C < 1 || y_type < 0 || y_type > 2 || H > 32768 || W > 32768) return PGAN_EINVAL;
    if (B == 0) return PGAN_OK;
    if (!y || !q || !scale || ldq < C || !aligned(y, type_bytes(y_type)) || !aligned(scale, 4)) return PGAN_EINVAL;
    const long long pixels = 4LL * B * H * W, blocks = (pixels + 3) / 4;
    if (blocks > MAX_BLOCKS) return PGAN_EINVAL;
    return by_type(y_type, [&](auto t) {
        up_fold_q8_kernel<t.value><<<(unsigned)blocks, 256, 0, st>>>(static_cast<const typename Elem<t.value>::type*>(y), shift,
                                                                      static_cast<int8_t*>(q), ldq, scale, pixels, H, W, C);
    });
}

int pgan_up_fold(const void* y, int y_type, const float* shift, float* out, int B, int H, int W, int C, int act,
                 hipStream_t st) {
    if (B < 0 || H < 1 || W < 1 || C < 1 || y_type < 0 || y_type > 2 || act < 0 || act > 2 || H > 32768 || W > 32768)
        return PGAN_EINVAL;
    if (B == 0) return PGAN_OK;
    if (!y || !out || !aligned(y, type_bytes(y_type)) || !aligned(out, 4)) return PGAN_EINVAL;
    const long long pixels = 4LL * B * H * W;
    if (pixels > MAX_BLOCKS * 256 / C) return PGAN_EINVAL;
    const long long blocks = (pixels * C + 255) / 256;
    return by_type(y_type, [&](auto t) {
        up_fold_kernel<t.value><<<(unsigned)blocks, 256, 0, st>>>(static_cast<const typename Elem<t.value>::type*>(y), shift,
                                                                   out, pixels, H, W, C, act);
    });
}

}  // extern "C"
