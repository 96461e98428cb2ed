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
#include <algorithm>

#include "../../include/pgan_hip.h"
#include "pgan_common.h"

// each product and sum rounded by itself: codes are the same wherever the formulas are evaluated in fp32
#pragma clang fp contract(off)

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
// Global memory takes wide accesses on any border; these say so.
typedef float f32x4_4 __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x2_4 __attribute__((ext_vector_type(2), aligned(4)));
typedef int i32x4_2 __attribute__((ext_vector_type(4), aligned(2)));
typedef int i32x2_2 __attribute__((ext_vector_type(2), aligned(2)));
typedef int i32x2_1 __attribute__((ext_vector_type(2), aligned(1)));

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
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true));
}
// maximum over aligned groups of 2^log lanes, in every lane of the group
__device__ __forceinline__ uint32_t group_max(uint32_t v, int log) {
    if (log > 0) v = dpp_max<0xB1>(v);
    if (log > 1) v = dpp_max<0x4E>(v);
    if (log > 2) v = dpp_max<0x141>(v);
    if (log > 3) v = dpp_max<0x140>(v);
    if (log > 4) v = max(v, (uint32_t)__shfl_xor((int)v, 16, 64));
    if (log > 5) v = max(v, (uint32_t)__shfl_xor((int)v, 32, 64));
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
// The code of x is the low byte of x inv + 1.5 2^23: that sum's last place is 1, so it is rounded to a whole number (ties to
// the even one).  A row without a finite maximum has inv = 0: its elements have to be made 0 first (no_row).
__device__ __forceinline__ uint32_t code_of(float x, float inv) { return __builtin_bit_cast(uint32_t, x * inv + 12582912.f); }
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d, float inv) {
    return __builtin_amdgcn_perm(code_of(b, inv), code_of(a, inv), 0x0c0c0400) | __builtin_amdgcn_perm(code_of(d, inv), code_of(c, inv), 0x04000c0c);
}
template <int N>
__device__ __forceinline__ void no_row(float (&v)[N], float inv) {
    if (inv == 0.f) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = 0.f;
    }
}
// LeakyReLU: of x and its tenth the larger
__device__ __forceinline__ float slope(float x, bool lrelu) { return lrelu ? __builtin_fmaxf(x, x * PGAN_SLOPE) : x; }

// eight elements from p on; NT: read once, past the caches
template <int TYPE, bool NT = false>
__device__ __forceinline__ void load8(const typename Elem<TYPE>::type* p, float (&v)[8]) {
    if constexpr (TYPE == 0) {
        const f32x4_4* x = reinterpret_cast<const f32x4_4*>(p);
        const f32x4 a = NT ? __builtin_nontemporal_load(x) : x[0], b = NT ? __builtin_nontemporal_load(x + 1) : x[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = a[e];
            v[4 + e] = b[e];
        }
    } else {
        const i32x4_2* x = reinterpret_cast<const i32x4_2*>(p);
        const i32x4 a = NT ? __builtin_nontemporal_load(x) : *x;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (TYPE == 1) {
                v[2 * e] = __builtin_bit_cast(float, a[e] << 16);
                v[2 * e + 1] = __builtin_bit_cast(float, a[e] & (int)0xffff0000);
            } else {
                v[2 * e] = (float)__builtin_bit_cast(_Float16, (uint16_t)a[e]);
                v[2 * e + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)((uint32_t)a[e] >> 16));
            }
        }
    }
}
// as load8 of fewer than eight elements in a row, zeros behind them
template <int TYPE>
__device__ __forceinline__ void load_few(const typename Elem<TYPE>::type* p, int n, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? to_f32<TYPE>(p[e]) : 0.f;
}
__device__ __forceinline__ void store_codes(int8_t* p, const float (&v)[8], float inv) {
    *reinterpret_cast<i32x2_1*>(p) = i32x2_1{(int)four_codes(v[0], v[1], v[2], v[3], inv), (int)four_codes(v[4], v[5], v[6], v[7], inv)};
}

// ---- rows to codes ------------------------------------------------------------------------------------------------
// 2^log lanes a row, whose values stay in their registers between the maximum and the codes: 8 NIT each, K <= 8 NIT 2^log; a
// lane has R rows, to have more bytes on their way.  A lane takes eight neighbouring elements at a time, the one at the row's
// end its last eight, some of them its neighbour's too.  Bound by HBM (2 + 1 bytes an element of 16 bits; 16000 x 512: 6.2 us where
// the same rows are taken again, 7.1 in front of its product, 8.8 out of 650 MB of rows in turn, 2.8 TB/s; launch and one trip to
// memory are half of it).
template <int TYPE, int NIT, int R>
__global__ __launch_bounds__(256) void quant_rows_kernel(const typename Elem<TYPE>::type* __restrict__ x, long long ldx,
                                                         int8_t* __restrict__ q, long long ldq, float* __restrict__ scale,
                                                         long long rows, int K, int lrelu, int log) {
    const long long row0 = ((long long)blockIdx.x * (256 >> log) + (threadIdx.x >> log)) * R;
    const int l = threadIdx.x & ((1 << log) - 1);
    if (row0 >= rows) return;        // whole groups of 2^log lanes
    float v[R][NIT][8];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const typename Elem<TYPE>::type* xr = x + (row0 + r < rows ? row0 + r : row0) * ldx;
#pragma unroll
        for (int it = 0; it < NIT; ++it) {
            const int k = ((it << log) + l) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[r][it][e] = 0.f;
            if (K < 8) load_few<TYPE>(xr, K, v[r][it]);
            else if (k < K) load8<TYPE>(xr + min(k, K - 8), v[r][it]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        uint32_t mx = 0;
#pragma unroll
        for (int it = 0; it < NIT; ++it)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[r][it][e] = slope(v[r][it][e], lrelu);
                mx = max(mx, magnitude(v[r][it][e]));
            }
        const RowScale rs = row_scale(group_max(mx, log));
        if (row0 + r >= rows) break;
        if (l == 0) scale[row0 + r] = rs.scale;
        int8_t* qr = q + (row0 + r) * ldq;
#pragma unroll
        for (int it = 0; it < NIT; ++it) {
            no_row(v[r][it], rs.inv);
            const int k = ((it << log) + l) * 8;
            if (K < 8) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < K) qr[e] = (int8_t)code_of(v[r][it][e], rs.inv);
            } else if (k < K) {
                store_codes(qr + min(k, K - 8), v[r][it], rs.inv);
            }
        }
    }
}

// Longer rows: one a block.  NIT > 0: the values stay in registers, 8 NIT of a thread (K <= 2048 NIT); 0: rows are read twice,
// the second time from the L2 or the memory-side cache.  From memory: 8192 x 8192 in bf16 43 us, 4.6 TB/s (read twice: 49), in fp32
// 65 us, 5.1 TB/s; read twice 8192 x 11008 in bf16 71 us, 3.8 TB/s, in fp32 125 us, 3.6 TB/s, 4096 x 28672 in bf16 102 us, 3.5 TB/s.
template <int TYPE, int NIT>
__global__ __launch_bounds__(256) void quant_long_rows_kernel(const typename Elem<TYPE>::type* __restrict__ x, long long ldx,
                                                              int8_t* __restrict__ q, long long ldq, float* __restrict__ scale,
                                                              long long rows, int K, int lrelu) {
    __shared__ uint32_t tops[4];
    const long long row = blockIdx.x;
    const typename Elem<TYPE>::type* xr = x + row * ldx;
    int8_t* qr = q + row * ldq;
    uint32_t mx = 0;
    const auto top = [&](float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = slope(v[e], lrelu);
            mx = max(mx, magnitude(v[e]));
        }
    };
    float kept[NIT > 0 ? NIT : 1][8];
    if constexpr (NIT > 0) {
#pragma unroll
        for (int i = 0; i < NIT; ++i)
            if (threadIdx.x * 8 + 2048 * i < K) load8<TYPE>(xr + min((int)threadIdx.x * 8 + 2048 * i, K - 8), kept[i]);
#pragma unroll
        for (int i = 0; i < NIT; ++i)
            if (threadIdx.x * 8 + 2048 * i < K) top(kept[i]);
    } else {
        for (int k = threadIdx.x * 8; k < K; k += 2048) {
            float v[8];
            load8<TYPE>(xr + min(k, K - 8), v);
            top(v);
        }
    }
    mx = group_max(mx, 6);
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = mx;
    __syncthreads();
    const RowScale rs = row_scale(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
    if (threadIdx.x == 0) scale[row] = rs.scale;
    if constexpr (NIT > 0) {
#pragma unroll
        for (int i = 0; i < NIT; ++i)
            if (threadIdx.x * 8 + 2048 * i < K) {
                no_row(kept[i], rs.inv);
                store_codes(qr + min((int)threadIdx.x * 8 + 2048 * i, K - 8), kept[i], rs.inv);
            }
    } else {
        for (int k = threadIdx.x * 8; k < K; k += 2048) {
            float v[8];
            load8<TYPE>(xr + min(k, K - 8), v);
            no_row(v, rs.inv);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = slope(v[e], lrelu);
            store_codes(qr + min(k, K - 8), v, rs.inv);
        }
    }
}

// ---- the product --------------------------------------------------------------------------------------------------
// A block of WT x WN waves (MW waves of all blocks on a SIMD at once) makes a tile of tokens x channels, a wave FT x FN tiles
// of 32 x 32 (i32 <- i8, 32 deep; channels are the matrix instruction's rows, so that a lane holds four neighbouring channels
// of one token).  Stages of GK bytes along K go from memory straight into a ring of D in LDS, without a stop in registers: a
// stage's place is refilled as soon as every wave has read its last step, which leaves the other D - 1 under way meanwhile.
// A wave waits for its own reads of a stage by their count and meets the others at a barrier, once a stage; the operands of
// a step of 32 are read from LDS between the products of the step before.
// Bound by the matrix instructions and the power they draw where K is long (8192 x 8192 x 8192: 458 us, 2400 Top/s, the
// rate of the library's product; 4096 x 4096 x 4096: 64 us, 2150 Top/s), by the results' way out where it is short (256000 x
// 128 x 1024: 95 us, 5.9 TB/s).  With stages that went through registers into one place of LDS 4096 x 4096 x 4096 took 77
// us and 2048 x 2048 x 2048 21 for 14; with all of a step's LDS reads before its products, and so the next stage's reads
// from memory waited for at once, 74 and 15; with results that stay in the caches 16000 x 512 x 4096 61 for 50 and
// 256000 x 128 x 1024 115 for 95: the kernel ends when they have left.
__device__ __forceinline__ i32x4 below(i32x4 v, int left) {        // the first `left` of 16 bytes, zero behind them
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int n = left - 4 * e;
        v[e] = n >= 4 ? v[e] : n <= 0 ? 0 : v[e] & ((1 << (8 * n)) - 1);
    }
    return v;
}

template <int TYPE>
__device__ __forceinline__ uint2 pack4(float a, float b, float c, float d) {
    using H = std::conditional_t<TYPE == 1, __bf16, _Float16>;
    typedef H h2 __attribute__((ext_vector_type(2)));
    return uint2{__builtin_bit_cast(uint32_t, h2{(H)a, (H)b}), __builtin_bit_cast(uint32_t, h2{(H)c, (H)d})};
}
// 16 bytes of a row, of which `left` elements lie inside it
template <class Y>
__device__ __forceinline__ void put16(Y* to, i32x4 v, int left) {
    constexpr int PER = 16 / (int)sizeof(Y);
    if (left >= PER) {
        *reinterpret_cast<i32x4_2*>(to) = v;
        return;
    }
    const Y* h = reinterpret_cast<const Y*>(&v);
#pragma unroll
    for (int e = 0; e < PER; ++e)
        if (e < left) to[e] = h[e];
}

// what a wave's lanes wrote to LDS is seen by its other lanes
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

struct GemmArgs {
    const int8_t* q;
    const float* qs;
    const int8_t* w;
    const float* ws;
    const float* bias;
    void* y;
    long long ldq, ldw, ldy, T;
    int N, K;
    unsigned tt, tn, band;      // tiles along the tokens and along the channels, channel tiles of a band
};

// Tile of a block: blocks go round the eight dies, each of which gets a run of neighbouring tiles -- bands of eight channel
// tiles, token tile by token tile -- so that what it reads stays in its L2.
__device__ __forceinline__ void tile_of(const GemmArgs& a, unsigned& tt, unsigned& tn) {
    const unsigned tiles = a.tt * a.tn, per = tiles / 8, rest = tiles % 8, die = blockIdx.x % 8;
    const unsigned id = die * per + min(die, rest) + blockIdx.x / 8;
    const unsigned band = id / (a.band * a.tt), in = id - band * a.band * a.tt, wide = min(a.band, a.tn - band * a.band);
    tt = in / wide;
    tn = band * a.band + in - tt * wide;
}

// waits until at most VM of the wave's memory operations are under way and all its LDS reads have come back
template <int VM>
__device__ __forceinline__ void wait_for() {
    __builtin_amdgcn_s_waitcnt((VM & 15) | 7 << 4 | (VM >> 4) << 14);
}

// 16 bytes a lane from `at` + `same` (the wave's) bytes into `from` to LDS: `to` + 16 * lane, without a stop in registers
__device__ __forceinline__ void read_to_lds(__amdgpu_buffer_rsrc_t from, char* to, int at, int same) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef __attribute__((address_space(3))) void lds_void;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_void*)to, 16, at, same, 0, 0);
#endif
}

template <int FT, int FN, int WT, int WN, int GK, int D, int MW, int TYPE>
__global__ __launch_bounds__(64 * WT * WN, MW) void gemm_q8_kernel(const GemmArgs a) {
    using Y = typename Elem<TYPE>::type;
    constexpr int NW = WT * WN, NT = 64 * NW, BT = 32 * FT * WT, BN = 32 * FN * WN;
    constexpr int RR = 1024 / GK, CH = GK / 16;          // rows of a wave's read, 16-byte chunks of a stage's row
    constexpr int SH = GK == 64 ? 2 : 1;                 // rows that 64 banks hold: 1 << SH
    constexpr int PX = BT / RR / NW, PW = BN / RR / NW, P = PX + PW;      // reads of a wave a stage, RR rows each
    static_assert(PX * RR * NW == BT && PW * RR * NW == BN && (D - 1) * P < 64 && NW % 2 == 0, "whole reads");
    constexpr int STAGE = (BT + BN) * GK;
    constexpr int FO = FN < 2 ? FN : 2;                  // channel tiles whose results leave together
    constexpr int YROW = 32 * FO * (int)sizeof(Y) + 16;  // a wave's row of results in LDS, 16 bytes apart
    constexpr int JO = TYPE == 0 || FT < 2 ? 1 : 2;      // token tiles
    constexpr int OUT = 32 * JO * YROW * WT * WN;
    constexpr int BYTES = D * STAGE > OUT ? D * STAGE : OUT;
    __shared__ __attribute__((aligned(16))) char mem[BYTES];
    __shared__ __attribute__((aligned(16))) float sws[BN], sbias[BN], sqs[BT];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wt = wave / WN, wn = wave % WN;
    unsigned tt, tn;
    tile_of(a, tt, tn);
    const long long t0 = (long long)tt * BT;
    const int n0 = (int)tn * BN, K = a.K, stages = (K + GK - 1) / GK;
    const int trows = (int)(a.T - t0 < BT ? a.T - t0 : BT), nrows = min(a.N - n0, BN);
    // the scales come first
    static_assert(BN <= NT && BT <= NT, "one scale a thread");
    const int sn = n0 + min(tid, nrows - 1);
    const float vws = a.ws[sn], vbias = a.bias ? a.bias[sn] : 0.f, vqs = a.qs[t0 + min(tid, trows - 1)];
    // A wave's read takes GK bytes of RR rows.  Chunk c of row r lies in LDS at r * CH + (c ^ ((r >> SH) % CH)): the 16 rows
    // that a quarter wave reads one chunk of then lie in different banks.  Rows past the end repeat the last one;
    // what they give is not stored.
    const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(a.q + t0 * a.ldq), 0, 0x7fffffff, 0x00020000);
    const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(a.w + (long long)n0 * a.ldw), 0, 0x7fffffff, 0x00020000);
    const int chunk = ((lane & (CH - 1)) ^ ((RR * wave + lane / CH) >> SH & (CH - 1))) * 16;       // the same for all of a lane's rows
    int xo[PX], wo[PW];
#pragma unroll
    for (int i = 0; i < PX; ++i) xo[i] = min((wave + NW * i) * RR + lane / CH, trows - 1) * (int)a.ldq + chunk;
#pragma unroll
    for (int i = 0; i < PW; ++i) wo[i] = min((wave + NW * i) * RR + lane / CH, nrows - 1) * (int)a.ldw + chunk;
    const int last = (K + 15) / 16 * 16 - 16 - chunk;        // of a stage's first byte, so that a row's last 16 bytes are read at most
    // one of the P reads of a stage; WHOLE: no place of the stage lies past K
    const auto fetch = [&](auto whole, int st, int i) {
        char* to = mem + st % D * STAGE + ((i < PX ? 0 : BT * GK) + (wave + NW * (i < PX ? i : i - PX)) * 1024);
        const int at = whole.value ? st * GK : 0, more = whole.value ? 0 : min(st * GK, last);
        if (i < PX) read_to_lds(xr, to, xo[i] + more, at);
        else read_to_lds(wr, to, wo[i - PX] + more, at);
    };
    const int at = (lane & 31) * GK + ((lane >> 5) ^ ((lane >> SH) & (CH - 1))) * 16;      // of step 0 in 32 rows; step s: ^ 32 s
    i32x4 fw[2][FN], fx[2][FT];
    // one of the FN + FT operands of a step, in the order in which they are needed
    const auto read = [&](int st, int s, int r) {
        const char* from = mem + st % D * STAGE + (at ^ 32 * s);
        if (r == 0 || r > FT) fw[s & 1][r == 0 ? 0 : r - FT] = *reinterpret_cast<const i32x4*>(from + (BT + (wn * FN + (r == 0 ? 0 : r - FT)) * 32) * GK);
        else fx[s & 1][r - 1] = *reinterpret_cast<const i32x4*>(from + (wt * FT + r - 1) * 32 * GK);
    };
    i32x16 acc[FN][FT];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FT; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
    const auto in_order = [] { __builtin_amdgcn_sched_barrier(0); };
    const auto meet = [] {
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    using std::bool_constant;
#pragma unroll
    for (int st = 0; st < D; ++st)
        if (st < stages)
#pragma unroll
            for (int i = 0; i < P; ++i) fetch(bool_constant<false>{}, st, i);
    if (tid < BN) {
        sws[tid] = vws;
        sbias[tid] = vbias;
    }
    if (tid < BT) sqs[tid] = vqs;
    if (D <= stages) wait_for<(D - 1) * P>();
    else wait_for<0>();
    meet();
#pragma unroll
    for (int r = 0; r < FN + FT; ++r) read(0, 0, r);
    // A stage's products, and between them the reads of the next step's operands and of stage st + D.  WHAT: 0 that is a whole
    // stage, 1 it is the last, 2 there is none, 3 nor a next one.
    const auto stage = [&](auto what, int st) {
        constexpr int WHAT = what.value, STEPS = GK / 32, NM = FN * FT, H = NM < 2 ? 1 : NM / 2;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const bool end = s + 1 == STEPS, more = !end || WHAT < 3;
            if (end && more) {      // every wave's part of the next stage is there, and every wave has read this one
                if (WHAT < 2 || st + D <= stages) wait_for<(D - 2) * P>();
                else wait_for<0>();
                meet();
            }
            if (WHAT == 3 && st * GK + 32 * s + 32 > K) {      // what stands past K does not count
#pragma unroll
                for (int i = 0; i < FN; ++i) fw[s & 1][i] = below(fw[s & 1][i], K - st * GK - 32 * s - 16 * (lane >> 5));
            }
            in_order();
#pragma unroll
            for (int n = 0; n < NM; ++n) {
                const int i = n / FT, j = n % FT;
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[s & 1][i], fx[s & 1][j], acc[i][j], 0, 0, 0);
                in_order();
                // LDS is read before it is written to: the compiler lets no read of it pass a write from memory
                if (more && n < H)
#pragma unroll
                    for (int r = n * (FN + FT) / H; r < (n + 1) * (FN + FT) / H; ++r) read(end ? st + 1 : st, end ? 0 : s + 1, r);
                in_order();
                if (WHAT < 2 && end && n >= NM - H)
#pragma unroll
                    for (int f = (n - NM + H) * P / H; f < (n - NM + H + 1) * P / H; ++f) fetch(bool_constant<WHAT == 0>{}, st + D, f);
                in_order();
            }
        }
    };
    using std::integral_constant;
    int st = 0;
    for (; st < stages - D - 1; ++st) stage(integral_constant<int, 0>{}, st);
    if (st < stages - D) stage(integral_constant<int, 1>{}, st++);
    for (; st < stages - 1; ++st) stage(integral_constant<int, 2>{}, st);
    stage(integral_constant<int, 3>{}, st);
    __syncthreads();
    // (In 16 bits, tokens 16 to 31 keep the two eights of every 16 bytes the other way round: a store's 32 lanes then touch
    // all 64 banks once.)
    // The results of 32 tokens at a time pass through the wave's part of LDS, to leave as whole lines of y's rows.
    // channel (within 32): e % 4 + 8 (e / 4) + 4 (lane / 32); token: lane % 32
    char* own = mem + wave * 32 * JO * YROW;
    constexpr int PER = 16 / (int)sizeof(Y), LANES = 32 * FO / PER;      // channels and lanes of a 16-byte row stretch
    const bool whole = trows == BT && nrows == BN;
#pragma unroll
    for (int io = 0; io < FN; io += FO) {
        const int wc0 = (wn * FN + io) * 32;
#pragma unroll
        for (int jo = 0; jo < FT; jo += JO) {
            const int tr = (wt * FT + jo) * 32;
            float st[JO];
#pragma unroll
            for (int j = 0; j < JO; ++j) st[j] = sqs[tr + 32 * j + (lane & 31)];
#pragma unroll
            for (int i = 0; i < FO; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int ch = 32 * i + 8 * g + 4 * (lane >> 5);
                    const f32x4 ws = *reinterpret_cast<const f32x4*>(sws + wc0 + ch), bs = *reinterpret_cast<const f32x4*>(sbias + wc0 + ch);
#pragma unroll
                    for (int j = 0; j < JO; ++j) {
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf((float)acc[io + i][jo + j][4 * g + e] * st[j], ws[e], bs[e]);
                        char* to = own + (32 * j + (lane & 31)) * YROW;
                        if constexpr (TYPE == 0) *reinterpret_cast<f32x4*>(to + ch * 4) = f32x4{v[0], v[1], v[2], v[3]};
                        else *reinterpret_cast<uint2*>(to + (ch * 2 ^ (lane & 16) / 2)) = pack4<TYPE>(v[0], v[1], v[2], v[3]);
                    }
                }
            wave_sync();
            Y* to = static_cast<Y*>(a.y) + (t0 + tr + lane / LANES) * a.ldy + n0 + wc0 + lane % LANES * PER;
            const char* from = own + lane / LANES * YROW + lane % LANES * 16;
            // 16 bytes of row r + lane / LANES; rows 16 to 31 of 32 hold their eights the other way round
            const auto piece = [&](int r) {
                const i32x4 v = *reinterpret_cast<const i32x4*>(from + r * YROW);
                return TYPE != 0 && (r & 16) ? i32x4{v[2], v[3], v[0], v[1]} : v;
            };
            if (whole) {
#pragma unroll
                for (int r = 0; r < 32 * JO; r += 64 / LANES) __builtin_nontemporal_store(i32x4_2(piece(r)), reinterpret_cast<i32x4_2*>(to + r * a.ldy));
            } else {
                for (int r = 0; r < 32 * JO; r += 64 / LANES)
                    if (tr + r + lane / LANES < trows) put16(to + r * a.ldy, piece(r), nrows - wc0 - lane % LANES * PER);
            }
            wave_sync();
        }
    }
}

// ---- the product for few tiles ------------------------------------------------------------------------------------
// A block makes 32 tokens x 32 channels, its WV waves share K and add up their sums (whole numbers: any order) in LDS.
// Channels come straight from memory into the matrix instruction's registers, every line of them by one wave.  X >= 0: the
// block makes the tokens' codes itself, a lane parts of RW rows -- every block all of them, which for few of them takes less time
// than a launch of its own -- while its first channels are on their way; X < 0: it reads codes.  Bound by the launch
// (1 x 128 x 8192: 3.7 us in a graph), then by the channels' bytes (1 x 8192 x 8192: 15 us, 4.5 TB/s).
struct FewArgs {
    GemmArgs g;
    const void* x;
    long long ldx;
    int lrelu, log;         // 2^log lanes make a row's codes, 512 elements at a time
};
template <int X, int WV, int RW, int TYPE>
__global__ __launch_bounds__(64 * WV) void gemm_few_kernel(const FewArgs f) {
    using Y = typename Elem<TYPE>::type;
    using XE = typename Elem<X < 0 ? 0 : X>::type;
    extern __shared__ __attribute__((aligned(16))) char few[];
    const GemmArgs& a = f.g;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int K = a.K, T = (int)min(a.T - blockIdx.y * 32LL, 32LL), N = a.N, end = (K + 15) / 16 * 16 - 16;    // a row's last 16 bytes
    const long long t0 = blockIdx.y * 32LL;
    const int n0 = blockIdx.x * 32, half = lane >> 5, stride = (K + 31) / 32 * 32 + 16;
    const int steps = (K + 31) / 32, s0 = wave * steps / WV, s1 = (wave + 1) * steps / WV;
    const int8_t* wr = a.w + (long long)min(n0 + (lane & 31), N - 1) * a.ldw;
    // Four steps (a line of each row) at a time.  A load of all lanes takes another step of every fourth row: were it the same
    // one, all 32 rows' lines would be asked for the same 32 bytes, which the L1 serves one after the other.  in_order()
    // turns a lane's four back.
    const auto four = [&](const int8_t* from, int s, i32x4 (&v)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const i32x4*>(from + min((s + ((i + lane) & 3)) * 32 + 16 * half, end));
    };
    const auto in_order = [&](i32x4 (&v)[4]) {
        const i32x4 a = v[0], b = v[1], c = v[2], d = v[3];
        const bool one = lane & 1, two = lane & 2;
        const i32x4 e = one ? d : a, f = one ? a : b, g = one ? b : c, h = one ? c : d;
        v[0] = two ? g : e;
        v[1] = two ? h : f;
        v[2] = two ? e : g;
        v[3] = two ? f : h;
    };
    i32x4 cur[4], nxt[4];
    four(wr, s0, cur);
    float ws[4], bs[4];         // of the four channels whose sums this lane ends
    const int ch = n0 + 8 * wave + 4 * half;
    if (wave < 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            ws[e] = a.ws[min(ch + e, N - 1)];
            bs[e] = a.bias ? a.bias[min(ch + e, N - 1)] : 0.f;
        }
    }
    __shared__ float scales[32];
    if constexpr (X >= 0) {
        const XE* x = static_cast<const XE*>(f.x);
        float v[RW][8];
        uint32_t mx[RW];
#pragma unroll
        for (int r = 0; r < RW; ++r) mx[r] = 0;
        const int l8 = (lane & ((1 << f.log) - 1)) * 8;
        const auto row_of = [&](int r) { return ((wave + WV * r) << (6 - f.log)) + (lane >> f.log); };
        const auto part = [&](int k0) {     // up to 512 elements of each of the wave's rows, a row's last eight at its end
#pragma unroll
            for (int r = 0; r < RW; ++r) {
                const XE* xr = x + (long long)row_of(r) * f.ldx;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[r][e] = 0.f;
                if (row_of(r) >= T || k0 + l8 >= K) continue;
                if (K < 8) load_few<X < 0 ? 0 : X>(xr, K, v[r]);
                else load8<X < 0 ? 0 : X>(xr + min(k0 + l8, K - 8), v[r]);
            }
#pragma unroll
            for (int r = 0; r < RW; ++r)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[r][e] = slope(v[r][e], f.lrelu);
        };
        for (int k0 = 0; k0 < K; k0 += 512) {
            part(k0);
#pragma unroll
            for (int r = 0; r < RW; ++r)
#pragma unroll
                for (int e = 0; e < 8; ++e) mx[r] = max(mx[r], magnitude(v[r][e]));
        }
        float inv[RW];
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            const RowScale rs = row_scale(group_max(mx[r], f.log));
            inv[r] = rs.inv;
            if (l8 == 0 && row_of(r) < T) scales[row_of(r)] = rs.scale;
        }
        for (int k0 = 0; k0 < K; k0 += 512) {
            if (K > 512) part(k0);
#pragma unroll
            for (int r = 0; r < RW; ++r)
                if (row_of(r) < T && k0 + l8 < K) {
                    no_row(v[r], inv[r]);
                    store_codes(reinterpret_cast<int8_t*>(few) + row_of(r) * stride + (K < 8 ? 0 : min(k0 + l8, K - 8)), v[r], inv[r]);
                }
        }
    } else {
        if (tid < 32) scales[tid] = a.qs[t0 + min(tid, T - 1)];
    }
    __syncthreads();
    const int t = lane & 31, row = min(t, T - 1);      // rows past the end repeat the last one; what they give is not stored
    i32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0;
    const int8_t* xr = X < 0 ? a.q + (t0 + row) * a.ldq : nullptr;
    i32x4 tok[4], more[4];
    if constexpr (X < 0) four(xr, s0, tok);
    for (int s = s0; s < s1; s += 4) {
        if (s + 4 < s1) {
            four(wr, s + 4, nxt);
            if constexpr (X < 0) four(xr, s + 4, more);
        }
        in_order(cur);
        if constexpr (X < 0) {
            in_order(tok);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) tok[i] = *reinterpret_cast<const i32x4*>(few + row * stride + min((s + i) * 32 + 16 * half, end));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (s + i < s1) {
                if ((s + i) * 32 + 32 > K) cur[i] = below(cur[i], K - (s + i) * 32 - 16 * half);
                acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(cur[i], tok[i], acc, 0, 0, 0);
            }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            cur[i] = nxt[i];
            if constexpr (X < 0) tok[i] = more[i];
        }
    }
    __syncthreads();
    i32x4* sums = reinterpret_cast<i32x4*>(few);       // [wave][four channels][lane]
#pragma unroll
    for (int g = 0; g < 4; ++g) sums[(wave * 4 + g) * 64 + lane] = i32x4{acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
    __syncthreads();
    if (wave >= 4 || t >= T) return;
    i32x4 sum = sums[wave * 64 + lane];
#pragma unroll
    for (int w = 1; w < WV; ++w) sum += sums[(w * 4 + wave) * 64 + lane];
    const float st = scales[t];
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf((float)sum[e] * st, ws[e], bs[e]);
    Y* to = static_cast<Y*>(a.y) + (t0 + t) * a.ldy + ch;
    if (ch + 4 <= N) {
        if constexpr (TYPE == 0) *reinterpret_cast<f32x4_4*>(to) = f32x4_4{v[0], v[1], v[2], v[3]};
        else *reinterpret_cast<i32x2_2*>(to) = __builtin_bit_cast(i32x2_2, pack4<TYPE>(v[0], v[1], v[2], v[3]));
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (ch + e < N) to[e] = from_f32<TYPE>(v[e]);
    }
}

// ---- the fold -----------------------------------------------------------------------------------------------------
// y: one row of 4 x 4 taps x C channels for each of B x H x W pixels; output pixel (oh, ow) of 2H x 2W is the sum of the
// (up to) four taps (kh, kw) of pixels (ih, iw) with oh = 2 ih + kh - 1, ow = 2 iw + kw - 1.  An even row takes tap 1 of
// its own input row and tap 3 of the one before, an odd row tap 2 of its own and tap 0 of the one after; so do columns.
struct Taps {
    long long at[2][2];     // first element of the tap's channels, -1: outside
};
__device__ __forceinline__ Taps taps_of(unsigned pix, int H, int W, int C) {
    const unsigned W2 = 2 * W, H2 = 2 * H;
    const unsigned line = pix / W2, b = line / H2;
    const int ow = (int)(pix - line * W2), oh = (int)(line - b * H2);
    const int ih = oh >> 1, iw = ow >> 1;
    const int h2 = oh & 1 ? ih + 1 : ih - 1, w2 = ow & 1 ? iw + 1 : iw - 1;
    const int ka = oh & 1 ? 2 : 1, kb = oh & 1 ? 0 : 3, la = ow & 1 ? 2 : 1, lb = ow & 1 ? 0 : 3;
    const bool hok = h2 >= 0 && h2 < H, wok = w2 >= 0 && w2 < W;
    const long long ra = ((long long)b * H + ih) * W, rb = ((long long)b * H + h2) * W;
    Taps t;
    t.at[0][0] = ((ra + iw) * 16 + ka * 4 + la) * C;
    t.at[1][0] = hok ? ((rb + iw) * 16 + kb * 4 + la) * C : -1;
    t.at[0][1] = wok ? ((ra + w2) * 16 + ka * 4 + lb) * C : -1;
    t.at[1][1] = hok && wok ? ((rb + w2) * 16 + kb * 4 + lb) * C : -1;
    return t;
}
// of the eight channels from c on, or of the only n < 8; NT: taps read past the caches
template <int TYPE, bool NT = true>
__device__ __forceinline__ void fold8(const typename Elem<TYPE>::type* y, const Taps& t, int c, int n, const float* shift, float (&v)[8]) {
    float p[2][2][8];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) p[i][j][e] = 0.f;
            if (t.at[i][j] < 0) continue;
            if (n < 8) load_few<TYPE>(y + t.at[i][j], n, p[i][j]);
            else load8<TYPE, NT>(y + t.at[i][j] + c, p[i][j]);
        }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (p[0][0][e] + p[1][0][e]) + (p[0][1][e] + p[1][1][e]);
    if (shift) {
        float sh[8];
        if (n < 8) load_few<0>(shift, n, sh);
        else load8<0>(shift + c, sh);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += sh[e];
    }
}
__device__ __forceinline__ float activate(float o, int act) {
    if (act == 1) return 1.f / (1.f + expf(-o));
    if (act == 2) return tanhf(o);
    return o;
}

struct FoldArgs {
    const float* shift;
    int8_t* q;
    float* scale;           // of codes
    float* out;             // or fp32 results
    long long ldq;
    unsigned pixels;
    int H, W, C, act, log;
};

// 2^log lanes an output pixel, eight neighbouring channels each, the last lane the pixel's last eight.  Every input value goes
// to exactly one output: nothing is read twice.  Bound by HBM (codes of 1000 x 16 x 16 x 64: 594 MB in 108 us, 5.5 TB/s; the
// codes past the caches too: 104, but the next product then waits for them, a thousand alignments drawn 600 us for 590).
template <int TYPE, bool Q8>
__global__ __launch_bounds__(256) void up_fold_kernel(const typename Elem<TYPE>::type* __restrict__ y, const FoldArgs a) {
    const unsigned pix = blockIdx.x * (256u >> a.log) + (threadIdx.x >> a.log);
    const int l = threadIdx.x & ((1 << a.log) - 1), C = a.C, c = C < 8 ? 0 : min(l * 8, C - 8);
    if (pix >= a.pixels) return;        // whole groups of 2^log lanes
    const Taps t = taps_of(pix, a.H, a.W, C);
    const bool some = l * 8 < C;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (some) fold8<TYPE>(y, t, c, C, a.shift, v);
    if constexpr (Q8) {
        uint32_t mx = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = slope(v[e], true);
            mx = max(mx, magnitude(v[e]));
        }
        const RowScale rs = row_scale(group_max(mx, a.log));
        if (l == 0) a.scale[pix] = rs.scale;
        no_row(v, rs.inv);
        int8_t* qr = a.q + (long long)pix * a.ldq;
        if (C < 8) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < C) qr[e] = (int8_t)code_of(v[e], rs.inv);
        } else if (some) {
            store_codes(qr + c, v, rs.inv);
        }
    } else {
        float* o = a.out + (long long)pix * C;
        if (C < 8) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < C) o[e] = activate(v[e], a.act);
        } else if (some) {
#pragma unroll
            for (int e = 0; e < 8; e += 4)
                *reinterpret_cast<f32x4_4*>(o + c + e) =
                    f32x4_4{activate(v[e], a.act), activate(v[e + 1], a.act), activate(v[e + 2], a.act), activate(v[e + 3], a.act)};
        }
    }
}

// More than 512 channels: one output pixel a wave, codes in two passes, of which only the second reads past the caches: 200 x 8 x
// 8 x 700 in bf16 101 us (133 with both past them, 103 with neither), in fp32 157 (249, 146), 16 x 16 x 16 x 8000 in bf16 402 (446,
// 457).  HBM and the second read of the taps: 3.2 TB/s of needed bytes where 400 x 8 x 8 x 512 in one pass makes 5.5.
template <int TYPE, bool Q8>
__global__ __launch_bounds__(256) void up_fold_wide_kernel(const typename Elem<TYPE>::type* __restrict__ y, const FoldArgs a) {
    const unsigned pix = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int l8 = (threadIdx.x & 63) * 8, C = a.C;
    if (pix >= a.pixels) return;
    const Taps t = taps_of(pix, a.H, a.W, C);
    float v[8];
    if constexpr (Q8) {
        uint32_t mx = 0;
        for (int c = l8; c < C; c += 512) {
            fold8<TYPE, false>(y, t, min(c, C - 8), C, a.shift, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = max(mx, magnitude(slope(v[e], true)));
        }
        const RowScale rs = row_scale(group_max(mx, 6));
        for (int c = l8; c < C; c += 512) {
            fold8<TYPE>(y, t, min(c, C - 8), C, a.shift, v);
            no_row(v, rs.inv);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = slope(v[e], true);
            store_codes(a.q + (long long)pix * a.ldq + min(c, C - 8), v, rs.inv);
        }
        if (l8 == 0) a.scale[pix] = rs.scale;
    } else {
        for (int c = l8; c < C; c += 512) {
            fold8<TYPE>(y, t, min(c, C - 8), C, a.shift, v);
            float* o = a.out + (long long)pix * C + min(c, C - 8);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = activate(v[e], a.act);
        }
    }
}

// One channel: a lane an input pixel, for the 2 x 2 output pixels on it.  It reads what its column gives them -- taps of row 3
// from the pixel above, 1 and 2 of its own, 0 of the one below, four at a time -- sums them along the column, and takes from its left and right neighbours their sums of column 3 and 0.  The
// first and last lane of a wave, whose neighbour is in another wave, make that neighbour's sums themselves.  Bound by HBM
// (1000 x 32 x 32: 49 MB in 11 us; tap by tap 32).
template <int TYPE>
__device__ __forceinline__ void load_taps(const typename Elem<TYPE>::type* p, float (&v)[4]) {
    if constexpr (TYPE == 0) {
        const f32x4 x = *reinterpret_cast<const f32x4_4*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = x[e];
    } else {
        const i32x2_2 x = *reinterpret_cast<const i32x2_2*>(p);
        const uint16_t h[4] = {(uint16_t)x[0], (uint16_t)((uint32_t)x[0] >> 16), (uint16_t)x[1], (uint16_t)((uint32_t)x[1] >> 16)};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = to_f32<TYPE>(__builtin_bit_cast(typename Elem<TYPE>::type, h[e]));
    }
}
template <int TYPE>
__global__ __launch_bounds__(256) void up_fold_one_kernel(const typename Elem<TYPE>::type* __restrict__ y, const FoldArgs a) {
    const unsigned i = blockIdx.x * 256 + threadIdx.x, n = a.pixels / 4, at = min(i, n - 1);
    const int H = a.H, W = a.W, lane = threadIdx.x & 63;
    const unsigned line = at / W, b = line / H;
    const int iw = (int)(at - line * W), ih = (int)(line - b * H);
    const bool up = ih > 0, down = ih + 1 < H;
    const auto* t = y + (long long)at * 16;
    float r1[4], r2[4], r3[4] = {0.f, 0.f, 0.f, 0.f}, r0[4] = {0.f, 0.f, 0.f, 0.f};
    load_taps<TYPE>(t + 4, r1);
    load_taps<TYPE>(t + 8, r2);
    if (up) load_taps<TYPE>(t + 12 - 16 * (long long)W, r3);
    if (down) load_taps<TYPE>(t + 16 * (long long)W, r0);
    float e[4], o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        e[k] = r1[k] + r3[k];
        o[k] = r2[k] + r0[k];
    }
    const auto column = [&](const typename Elem<TYPE>::type* t, float& even, float& odd) {      // the sums of a neighbour's column
        even = to_f32<TYPE>(t[4]) + (up ? to_f32<TYPE>(t[12 - 16 * (long long)W]) : 0.f);
        odd = to_f32<TYPE>(t[8]) + (down ? to_f32<TYPE>(t[16 * (long long)W]) : 0.f);
    };
    float le = __shfl_up(e[3], 1, 64), lo = __shfl_up(o[3], 1, 64), re = __shfl_down(e[0], 1, 64), ro = __shfl_down(o[0], 1, 64);
    if (lane == 0 && iw > 0) column(t - 16 + 3, le, lo);
    if (lane == 63 && iw + 1 < W) column(t + 16, re, ro);
    if (i >= n) return;
    if (iw == 0) le = lo = 0.f;
    if (iw + 1 == W) re = ro = 0.f;
    const float sh = a.shift ? a.shift[0] : 0.f;
    const auto end = [&](float x) { return activate(a.shift ? x + sh : x, a.act); };
    float* to = a.out + ((long long)line * 4 * W + 2 * iw);
    *reinterpret_cast<f32x2_4*>(to) = f32x2_4{end(e[1] + le), end(e[2] + re)};
    *reinterpret_cast<f32x2_4*>(to + 2 * W) = f32x2_4{end(o[1] + lo), end(o[2] + ro)};
}

// threads of one launch stay below 2^32
constexpr long long MAX_BLOCKS = 0xffffff;
inline bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
inline int type_bytes(int type) { return type == 0 ? 4 : 2; }

constexpr long long MAX_STRIDE = 1 << 22;      // offsets of a tile's rows fit 31 bits
constexpr int MAX_ROW = 1 << 30;               // elements, so that a place in a row plus a block's stride does too

// lanes a row or an output pixel (as a power of two): eight elements each, all 64 for more than 256
inline int lanes_log(int C) {
    int log = 0;
    while (log < 6 && (8 << log) < C) ++log;
    return log;
}

constexpr int FEW = 32;
// waves of a block of a product of few tiles, and rows that they make the codes of at a time (512 elements of each)
inline int few_waves(int K) { return K >= 1024 ? 8 : 4; }
inline int few_rows(int K) { return few_waves(K) << (6 - lanes_log(K)); }
// Where the product's blocks make the codes themselves, each wave does so for RW times its share of few_rows(K); 0: rows to
// codes is a launch of its own.  launch_few takes RW from here, so that RW few_rows(K) >= T holds for what is launched.  They do
// where that takes a wave four loads a lane at most: us in one launch and in two, 16 x 512 x 1024 6.2 and 6.2, 8 x 700 x 1024 7.1
// and 7.2, 8 x 2048 x 1024 7.3 and 7.5, 32 x 128 x 8192 4.9 and 6.2, in a graph 8 x 1024 x 512 4.6 and 6.0, 12 x 1024 x 4096 5.8 and
// 5.8, 16 x 1024 x 4096 6.4 and 5.8 (called from a program, that is a launch less); past that 32 x 512 x 1024 9.1 and 6.2, 16 x 700
// x 1024 10.2 and 7.2, 1 x 4096 x 1024 10.2 and 9.1.
inline int few_coded(long long T, int K) {
    if (T < 1 || T > FEW || K < 1) return 0;
    for (int rw = 1; rw <= 4 && rw * ((K - 1) / 512 + 1) <= 4; rw *= 2)
        if (T <= rw * few_rows(K)) return rw;
    return 0;
}

template <int FT, int FN, int WT, int WN, int GK, int D, int MW, int TYPE>
void launch_gemm(GemmArgs a, hipStream_t st) {
    a.tn = (a.N + 32 * FN * WN - 1) / (32 * FN * WN);
    a.band = a.tn < 8 ? a.tn : 8;
    a.tt = (unsigned)((a.T + 32 * FT * WT - 1) / (32 * FT * WT));
    gemm_q8_kernel<FT, FN, WT, WN, GK, D, MW, TYPE><<<a.tt * a.tn, 64 * WT * WN, 0, st>>>(a);
}

template <class F>
inline int by_type(int type, F f) {
    switch (type) {
        case 0: f(std::integral_constant<int, 0>{}); break;
        case 1: f(std::integral_constant<int, 1>{}); break;
        default: f(std::integral_constant<int, 2>{}); break;
    }
    return pgan_launch_status();
}

// What an operand covers; outputs may not share memory with anything else of the call.
struct Span {
    const void* p;
    long long bytes;
    bool written;
};
inline Span rows_of(const void* p, long long rows, long long cols, long long ld, int size, bool written = false) {
    return Span{p, p ? ((rows - 1) * ld + cols) * size : 0, written};
}
template <int N>
bool apart(const Span (&s)[N]) {
    for (int i = 0; i < N; ++i)
        for (int j = i + 1; j < N; ++j) {
            if (!(s[i].written || s[j].written) || !s[i].bytes || !s[j].bytes) continue;
            const uintptr_t a = reinterpret_cast<uintptr_t>(s[i].p), b = reinterpret_cast<uintptr_t>(s[j].p);
            if (a < b + (uintptr_t)s[j].bytes && b < a + (uintptr_t)s[i].bytes) return false;
        }
    return true;
}

inline bool fold_fits(int type, int B, int H, int W, int C) {
    if (B < 0 || H < 1 || W < 1 || C < 1 || C > MAX_ROW || type < 0 || type > 2 || H > 32768 || W > 32768) return false;
    return B <= ((MAX_BLOCKS * 256) >> lanes_log(C)) / (4LL * H * W);
}
template <bool Q8>
int launch_fold(const void* y, int type, FoldArgs a, hipStream_t st) {
    a.log = lanes_log(a.C);
    const unsigned per = 256u >> a.log, blocks = a.pixels / per + (a.pixels % per != 0);
    return by_type(type, [&](auto t) {
        const auto* p = static_cast<const typename Elem<t.value>::type*>(y);
        if (a.C > 512) up_fold_wide_kernel<t.value, Q8><<<blocks, 256, 0, st>>>(p, a);
        else up_fold_kernel<t.value, Q8><<<blocks, 256, 0, st>>>(p, a);
    });
}

// up to 32 tokens x (of type X), or codes of any number (X < 0); false: no kernel makes the codes of so many
template <int X, int Y>
bool launch_few(const FewArgs& f, hipStream_t st) {
    const int K = f.g.K, codes = X < 0 ? 0 : (int)f.g.T * ((K + 31) / 32 * 32 + 16);
    const dim3 blocks((unsigned)((f.g.N + 31) / 32), X < 0 ? (unsigned)((f.g.T + 31) / 32) : 1u);
    // eight waves from K = 1024 on (us with 4, 8, 16: 1 x 8192 x 8192 16, 15, 15; 96 x 2048 x 2048 5.4, 4.8, 4.8; 64 x 4096 x
    // 8192 12.5, 13.3, 15.2; 1 x 512 x 4096 3.7, 3.9, -)
    const auto go = [&](auto waves, auto rows) {
        constexpr int WV = waves.value;
        gemm_few_kernel<X, WV, rows.value, Y><<<blocks, 64 * WV, std::max(codes, WV * 4096), st>>>(f);
        return true;
    };
    using std::integral_constant;
    constexpr integral_constant<int, 4> four;
    constexpr integral_constant<int, 8> eight;
    constexpr integral_constant<int, 1> one;
    if constexpr (X < 0) {
        return few_waves(K) == 8 ? go(eight, one) : go(four, one);
    } else {
        switch (few_waves(K) * 8 + few_coded(f.g.T, K)) {
            case 4 * 8 + 1: return go(four, one);
            case 4 * 8 + 2: return go(four, integral_constant<int, 2>{});
            case 4 * 8 + 4: return go(four, integral_constant<int, 4>{});
            case 8 * 8 + 1: return go(eight, one);
            case 8 * 8 + 2: return go(eight, integral_constant<int, 2>{});
            default: return false;
        }
    }
}

// Tiles of a product, tokens x channels; few: blocks of 32 x 32 whose waves share K
enum class Tiling { few, t128x32, t256x256, t128x256, t128x128, t128x64, t64x32, t64x64 };
inline Tiling tiling_of(long long T, int N, int K) {
    const auto tiles = [&](long long bt, long long bn) { return (T + bt - 1) / bt * ((N + bn - 1) / bn); };
    // how many in a hundred of the CUs that the last round of tiles takes along have one
    const auto fill = [&](long long bt, long long bn) { return tiles(bt, bn) * 100 / ((tiles(bt, bn) + 255) / 256 * 256); };
    // The larger the tile the fewer LDS reads a product takes; the smaller, the more blocks a CU has to hide one's results
    // behind another's products; and the last round of tiles should find a tile for most of the 256 CUs.  us in tiles of
    // 256 x 256 (eight waves, one block a CU), 128 x 256 (eight waves, two blocks), 128 x 128 (four blocks), 128 x 64,
    // 64 x 64, results in bf16:
    //   4096 x 4096 x 4096     63   74   83   82  102      16000 x 512 x 4096     53   47   50   62   86
    //   4096 x 2048 x 4096     36   40   45   45   58       4000 x 512 x 4096     15   14   15   17   21
    //   3000 x 4000 x 3000     43   59   51   51   59      64000 x 256 x 2048     82   69   65   85  116
    //   5000 x 2048 x 2000     28   31   28   29   36    256000 x 128 x 1024     118  106   96  127  173
    //   6000 x 1200 x 6000     68   59   63   71   94       9493 x 422 x 7069     82   75   83  111  107
    //   2500 x 2500 x 2500     31   25   25   33   31      10000 x 1000 x 1000    19   20   18   20   22
    //   1037 x 2288 x 5552     27   21   23   28   25       4000 x 2000 x 1000    24   17   17   14   17
    //   2000 x 8000 x 2000     73   54   55   42   54       2048 x 2048 x 2048    24   18   17   13   17
    //   1500 x 4000 x 1500     40   29   28   22   21       1944 x 1575 x 1304    21   14   15   12   12
    // and 1024000 x 64 x 16 takes 21 us in tiles of 128 x 32 (two waves), 43 in tiles of 128 x 128.  A product of few tiles
    // shares K among the waves of a block of 32 x 32 instead, one of somewhat more takes tiles of 64 x 32 (two waves): us in
    // 32 x 32, 64 x 32, 64 x 64
    //   64 x 4096 x 1024      7.3   9.3  11.1         704 x 4096 x 688     12.8  10.7  12.2
    //   512 x 4096 x 512      8.7   9.5  11.1        1024 x 4096 x 512     13.1  10.3  11.7
    //   512 x 512 x 512       3.9   4.2   4.3        1024 x 1024 x 512      5.6   5.0   5.3
    //                                                1024 x 2048 x 1024    12.4   8.1   7.6
    if (T <= FEW || tiles(64, 64) <= 64) return Tiling::few;
    if (N <= 32) return Tiling::t128x32;
    if (K >= 1024 && fill(256, 256) >= (K < 2048 ? 90 : 55)) return Tiling::t256x256;
    if (K > 256 && fill(128, 256) >= 70) return Tiling::t128x256;
    if (tiles(128, 128) >= 448) return Tiling::t128x128;
    if (tiles(128, 64) >= 320) return Tiling::t128x64;
    return tiles(64, 64) <= 128 ? Tiling::t64x32 : Tiling::t64x64;
}
// whether its launch has fewer than 2^32 threads
inline bool launch_holds(long long T, int N, int K) {
    const auto threads = [&](long long bt, long long bn, long long of) { return (T + bt - 1) / bt * ((N + bn - 1) / bn) * of < 1LL << 32; };
    switch (tiling_of(T, N, K)) {
        case Tiling::few: return threads(1LL << 40, 32, 512);       // along the channels; tokens are another dimension
        case Tiling::t128x32: return threads(128, 32, 128);
        case Tiling::t256x256: return threads(256, 256, 512);
        case Tiling::t128x256: return threads(128, 256, 512);
        case Tiling::t128x128: return threads(128, 128, 256);
        case Tiling::t128x64: return threads(128, 64, 256);
        case Tiling::t64x32: return threads(64, 32, 128);
        default: return threads(64, 64, 256);
    }
}

inline int gemm_args(const void* q, long long ldq, const float* q_scale, const void* w, long long ldw, const float* w_scale,
                     const float* bias, const void* y, int y_type, long long ldy, long long T, int N, int K) {
    if (T < 0 || N < 1 || K < 1 || K > 131072 || y_type < 0 || y_type > 2) return PGAN_EINVAL;
    if (T == 0) return PGAN_OK;
    if (!q || !q_scale || !w || !w_scale || !y || !aligned(q, 16) || !aligned(w, 16) || ldq % 16 || ldw % 16 || ldq < K
        || ldw < K || ldy < N || ldq > MAX_STRIDE || ldw > MAX_STRIDE || !aligned(y, type_bytes(y_type)))
        return PGAN_EINVAL;
    if (!apart({rows_of(y, T, N, ldy, type_bytes(y_type), true), rows_of(q, T, K, ldq, 1), rows_of(q_scale, 1, T, 0, 4),
                rows_of(w, N, K, ldw, 1), rows_of(w_scale, 1, N, 0, 4), rows_of(bias, 1, N, 0, 4)}))
        return PGAN_EINVAL;
    // fewer than 2^31 tokens and 2^28 channels, which keeps the counts of tiles inside 64 bits, and a launch that holds them
    if ((N + 31LL) / 32 > MAX_BLOCKS / 2 || T > MAX_BLOCKS / 2 * 256) return PGAN_EINVAL;
    return launch_holds(T, N, K) ? PGAN_OK : PGAN_EINVAL;
}

}  // namespace

extern "C" {

int pgan_quant_rows(const void* x, int x_type, long long ldx, void* q, long long ldq, float* scale, long long rows, int K,
                    int lrelu, hipStream_t st) {
    if (rows < 0 || K < 1 || K > MAX_ROW || x_type < 0 || x_type > 2) return PGAN_EINVAL;
    if (rows == 0) return PGAN_OK;
    if (!x || !q || !scale || !aligned(x, type_bytes(x_type)) || !aligned(scale, 4) || ldx < K || ldq < K) return PGAN_EINVAL;
    if (!apart({rows_of(x, rows, K, ldx, type_bytes(x_type)), rows_of(q, rows, K, ldq, 1, true), rows_of(scale, 1, rows, 0, 4, true)}))
        return PGAN_EINVAL;
    const int log = lanes_log(K);    // lanes a row
    // Rows of more than 1024 elements by a block: in a wave's registers 4096 x 4096 in bf16 took 14.9 us for 12.9, 8192 x 2048
    // 15.0 for 12.8, 300 x 2048 4.2 for 2.8, though 4000 x 1024 6.0 for 6.4.
    constexpr int LONG_ROW = 1024;
    // Rows a lane: two where there are enough of them (16000 x 512 in bf16: 9.3 us with one, 6.7 with two)
    const int R = K <= 1024 && rows >= 8192 ? 2 : 1;
    const long long groups = (rows + R - 1) / R, blocks = K > LONG_ROW ? rows : (groups + (256 >> log) - 1) / (256 >> log);
    if (blocks > MAX_BLOCKS) return PGAN_EINVAL;
    return by_type(x_type, [&](auto t) {
        constexpr int X = t.value;
        const auto go = [&](auto kernel, auto... more) {
            kernel<<<(unsigned)blocks, 256, 0, st>>>(static_cast<const typename Elem<X>::type*>(x), ldx, static_cast<int8_t*>(q), ldq,
                                                      scale, rows, K, lrelu, more...);
        };
        if (K > 8192) go(quant_long_rows_kernel<X, 0>);
        else if (K > 4096) go(quant_long_rows_kernel<X, 4>);
        else if (K > 2048) go(quant_long_rows_kernel<X, 2>);
        else if (K > LONG_ROW) go(quant_long_rows_kernel<X, 1>);
        else if (K > 512) R == 2 ? go(quant_rows_kernel<X, 2, 2>, log) : go(quant_rows_kernel<X, 2, 1>, log);
        else R == 2 ? go(quant_rows_kernel<X, 1, 2>, log) : go(quant_rows_kernel<X, 1, 1>, log);
    });
}

int pgan_gemm_q8(const void* q, long long ldq, const float* q_scale, const void* w, long long ldw, const float* w_scale,
                 const float* bias, void* y, int y_type, long long ldy, long long T, int N, int K, hipStream_t st) {
    const int rc = gemm_args(q, ldq, q_scale, w, ldw, w_scale, bias, y, y_type, ldy, T, N, K);
    if (rc || T == 0) return rc;
    return by_type(y_type, [&](auto t) {
        constexpr int Y = t.value;
        GemmArgs a{static_cast<const int8_t*>(q), q_scale, static_cast<const int8_t*>(w), w_scale, bias, y, ldq, ldw, ldy, T, N, K, 0, 0, 0};
        switch (tiling_of(T, N, K)) {
            case Tiling::few: launch_few<-1, Y>(FewArgs{a, nullptr, 0, 0, 0}, st); break;
            case Tiling::t128x32: launch_gemm<2, 1, 2, 1, 64, 2, 4, Y>(a, st); break;
            case Tiling::t256x256: launch_gemm<4, 2, 2, 4, 64, 4, 2, Y>(a, st); break;
            case Tiling::t128x256: launch_gemm<2, 2, 2, 4, 64, 3, 4, Y>(a, st); break;
            case Tiling::t128x128: launch_gemm<2, 2, 2, 2, 64, 2, 4, Y>(a, st); break;
            case Tiling::t128x64: launch_gemm<2, 1, 2, 2, 128, 2, 3, Y>(a, st); break;
            case Tiling::t64x32: launch_gemm<1, 1, 2, 1, 128, 4, 2, Y>(a, st); break;
            case Tiling::t64x64: launch_gemm<1, 1, 2, 2, 128, 3, 3, Y>(a, st); break;
        }
    });
}

int pgan_linear_q8_rows(long long T, int K) { return few_coded(T, K) * few_rows(K < 1 ? 1 : K); }

int pgan_linear_q8(const void* x, int x_type, long long ldx, void* q, long long ldq, float* q_scale, const void* w,
                   long long ldw, const float* w_scale, const float* bias, void* y, int y_type, long long ldy, long long T,
                   int N, int K, int lrelu, hipStream_t st) {
    const int ok = gemm_args(q, ldq, q_scale, w, ldw, w_scale, bias, y, y_type, ldy, T, N, K);
    if (ok || T == 0) return ok;
    if (x_type < 0 || x_type > 2 || !x || ldx < K || !aligned(x, type_bytes(x_type))
        || !apart({rows_of(x, T, K, ldx, type_bytes(x_type)), rows_of(y, T, N, ldy, type_bytes(y_type), true), rows_of(q, T, K, ldq, 1, true),
                   rows_of(q_scale, 1, T, 0, 4, true), rows_of(w, N, K, ldw, 1), rows_of(w_scale, 1, N, 0, 4), rows_of(bias, 1, N, 0, 4)}))
        return PGAN_EINVAL;
    if (few_coded(T, K)) {
        bool launched = false;
        const int rc = by_type(x_type, [&](auto xt) {
            (void)by_type(y_type, [&](auto t) {
                const GemmArgs a{nullptr, nullptr, static_cast<const int8_t*>(w), w_scale, bias, y, 0, ldw, ldy, T, N, K, 0, 0, 0};
                launched = launch_few<xt.value, t.value>(FewArgs{a, x, ldx, lrelu, lanes_log(K)}, st);
            });
        });
        return launched ? rc : PGAN_EINVAL;
    }
    const int rc = pgan_quant_rows(x, x_type, ldx, q, ldq, q_scale, T, K, lrelu, st);
    return rc ? rc : pgan_gemm_q8(q, ldq, q_scale, w, ldw, w_scale, bias, y, y_type, ldy, T, N, K, st);
}

int pgan_up_fold_q8(const void* y, int y_type, const float* shift, void* q, long long ldq, float* scale, int B, int H, int W,
                    int C, hipStream_t st) {
    if (!fold_fits(y_type, B, H, W, C)) return PGAN_EINVAL;
    if (B == 0) return PGAN_OK;
    if (!y || !q || !scale || ldq < C || !aligned(y, type_bytes(y_type)) || !aligned(scale, 4)) return PGAN_EINVAL;
    const long long pixels = 4LL * B * H * W;
    if (!apart({rows_of(y, 1, pixels * 4 * C, 0, type_bytes(y_type)), rows_of(shift, 1, C, 0, 4), rows_of(q, pixels, C, ldq, 1, true),
                rows_of(scale, 1, pixels, 0, 4, true)}))
        return PGAN_EINVAL;
    FoldArgs a{shift, static_cast<int8_t*>(q), scale, nullptr, ldq, (unsigned)pixels, H, W, C, 0, 0};
    return launch_fold<true>(y, y_type, a, st);
}

int pgan_up_fold(const void* y, int y_type, const float* shift, float* out, int B, int H, int W, int C, int act,
                 hipStream_t st) {
    if (!fold_fits(y_type, B, H, W, C) || act < 0 || act > 2) return PGAN_EINVAL;
    if (B == 0) return PGAN_OK;
    if (!y || !out || !aligned(y, type_bytes(y_type)) || !aligned(out, 4)) return PGAN_EINVAL;
    const long long pixels = 4LL * B * H * W;
    if (!apart({rows_of(y, 1, pixels * 4 * C, 0, type_bytes(y_type)), rows_of(shift, 1, C, 0, 4), rows_of(out, 1, pixels * C, 0, 4, true)}))
        return PGAN_EINVAL;
    FoldArgs a{shift, nullptr, nullptr, out, 0, (unsigned)pixels, H, W, C, act, 0};
    if (C == 1)
        return by_type(y_type, [&](auto t) {
            const auto* p = static_cast<const typename Elem<t.value>::type*>(y);
            up_fold_one_kernel<t.value><<<(a.pixels / 4 + 255) / 256, 256, 0, st>>>(p, a);
        });
    return launch_fold<false>(y, y_type, a, st);
}

}  // extern "C"
