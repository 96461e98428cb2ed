// AdamW over many tensors in one launch, its two states in 32 or in 8 bits (torch.optim.AdamW semantics; the reference
// steps its networks with torch.optim.Adam, src/train_wgan_v2.py:489-490,612,634).
//
//   m <- b1 m + (1 - b1) g        v <- b2 v + (1 - b2) g^2
//   p <- p (1 - lr wd) - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// States in 8 bits: blocks of 256 elements of a tensor, each with two power-of-two scales that bring the block's largest
// magnitudes into [128, 256); m and sqrt(v) are held as e4m3 codes (four exponent bits, three of mantissa) of the scaled
// value.  A power of two costs nothing of a floating code's relative precision and makes scaling exact.  Codes are rounded
// stochastically: at b2 = 0.999 a step changes v by 0.1 % or less while neighbouring codes are 6 to 12 % apart, so rounding
// to the nearest would leave v where it is for ever.  The random bits are a hash of (seed, step, tensor, place): a step is
// reproducible and nothing depends on the launch's shape.  A root that is not zero never becomes zero (its code is at least
// 1): a zero denominator beside an m that survived its own rounding would throw the parameter off by m / eps.  Rounding is without
// bias in what is held, m and the root, not in v, the root's square: over many steps of gradients of one variance v stands 4 %
// above what 32 bits give (b2 = 0.99: 3.9 %; at most 14 %: a step moves the root by d, codes are s apart, and rounding adds up to
// d s to v), and the root spreads by 15 % of itself (32 bits: 1.6 % at b2 = 0.999, 5 % at 0.99).  A state that is not finite is held as NaN, as it would poison the element in 32 bits too; it does not touch its block's scale.
//
// One launch for all tensors, as most of a network's are tiny: a block takes 2048 elements of one of them (a wave two blocks
// of 256 with 8-bit states, the second's reads under way while the first is computed).  Bound by HBM: 28 bytes an element
// with fp32 states (36 M elements: 172 us, 5.8 TB/s; a copy makes 4.86), 10 in bf16 with 8-bit ones (46 M elements: 94 us,
// 4.9 TB/s, hash and codes take almost as long), 26 tensors of 2.8 M elements 13 us.
#include <algorithm>
#include <vector>

#include "../../include/pgan_hip.h"
#include "pgan_common.h"

// Products and sums are rounded one by one, as the formulas are written: a code's rounding is then the same wherever the
// formulas are evaluated in fp32.  The kernels wait for memory either way.
#pragma clang fp contract(off)

namespace {

constexpr int AW_MAX = 40;          // tensors per launch: what fits the kernel arguments (4 KiB)
constexpr int AW_CHUNK = 2048;      // elements of a tensor per block of 256 threads
constexpr int AW_BLOCK = 256;       // elements that share a scale
constexpr long long AW_MOST = 0xffffff;      // blocks per launch (fewer than 2^32 threads)

struct AwTensor {
    void* p;
    const void* g;
    void* m;
    void* v;
    float* ms;
    float* rs;
    long long n;
    float size;                     // lr / (1 - b1^t); lr alone where the step count lives on the device
    float keep;                     // 1 - lr wd
    int types;                      // p type + 3 * g type
    int index;                      // number of the tensor in the caller's list
};
struct AwArgs {
    AwTensor t[AW_MAX];
    unsigned first[AW_MAX];         // first chunk of each tensor
    const int* step_dev;
    int n, step;
    float b1, c1, b2, c2, eps, gs, inv2;
    unsigned seed;
};

__device__ __forceinline__ uint32_t mix(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x6A09E667u;
    x = (x ^ (x >> 15)) * 0xBB67AE85u;
    return x ^ (x >> 16);
}

__device__ __forceinline__ float from16(uint16_t u, int type) {
    return type == 1 ? __builtin_bit_cast(float, (uint32_t)u << 16) : (float)__builtin_bit_cast(_Float16, u);
}
__device__ __forceinline__ uint16_t to16(float x, int type) {
    if (type == 1) {
        const uint32_t u = __builtin_bit_cast(uint32_t, x);
        return x != x ? (uint16_t)((u >> 16) | 0x40u) : (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
    }
    return __builtin_bit_cast(uint16_t, (_Float16)x);
}

// Four elements in one access, on any border (global memory takes them so); NT: past the caches.
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2_2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32_1 __attribute__((aligned(1)));
typedef float f32x4_4 __attribute__((ext_vector_type(4), aligned(4)));

template <bool NT>
__device__ __forceinline__ f32x4 get(const float* p) {
    const f32x4_4* q = reinterpret_cast<const f32x4_4*>(p);
    return NT ? __builtin_nontemporal_load(q) : *q;
}
template <bool NT>
__device__ __forceinline__ u32x2 get(const uint16_t* p) {
    const u32x2_2* q = reinterpret_cast<const u32x2_2*>(p);
    return NT ? __builtin_nontemporal_load(q) : *q;
}
template <bool NT>
__device__ __forceinline__ uint32_t get(const uint8_t* p) {
    const u32_1* q = reinterpret_cast<const u32_1*>(p);
    return NT ? __builtin_nontemporal_load(q) : *q;
}
template <bool NT>
__device__ __forceinline__ void put(float* p, f32x4_4 v) {
    f32x4_4* q = reinterpret_cast<f32x4_4*>(p);
    if constexpr (NT) __builtin_nontemporal_store(v, q);
    else *q = v;
}
template <bool NT>
__device__ __forceinline__ void put(uint16_t* p, u32x2_2 v) {
    u32x2_2* q = reinterpret_cast<u32x2_2*>(p);
    if constexpr (NT) __builtin_nontemporal_store(v, q);
    else *q = v;
}
template <bool NT>
__device__ __forceinline__ void put(uint8_t* p, uint32_t v) {
    u32_1* q = reinterpret_cast<u32_1*>(p);
    if constexpr (NT) __builtin_nontemporal_store(v, q);
    else *q = v;
}

// Four elements of a tensor: o (a lane's) past b, which is the same for the whole wave and stays in scalar registers.  VEC: one
// access, else those below n one by one.
template <int TYPE, bool VEC, bool NT>
__device__ __forceinline__ void load4(const void* src, long long b, int o, long long n, float (&v)[4]) {
    if constexpr (TYPE == 0) {
        const float* s = static_cast<const float*>(src) + b;
        if constexpr (VEC) {
            const f32x4 x = get<NT>(s + o);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = x[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = b + o + e < n ? s[o + e] : 0.f;
        }
    } else {
        const uint16_t* s = static_cast<const uint16_t*>(src) + b;
        if constexpr (VEC) {
            const u32x2 x = get<NT>(s + o);
            if constexpr (TYPE == 1) {
                v[0] = __builtin_bit_cast(float, x.x << 16);
                v[1] = __builtin_bit_cast(float, x.x & 0xffff0000u);
                v[2] = __builtin_bit_cast(float, x.y << 16);
                v[3] = __builtin_bit_cast(float, x.y & 0xffff0000u);
            } else {
                v[0] = from16((uint16_t)x.x, TYPE);
                v[1] = from16((uint16_t)(x.x >> 16), TYPE);
                v[2] = from16((uint16_t)x.y, TYPE);
                v[3] = from16((uint16_t)(x.y >> 16), TYPE);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = b + o + e < n ? from16(s[o + e], TYPE) : 0.f;
        }
    }
}
template <int TYPE, bool VEC, bool NT>
__device__ __forceinline__ void store4(void* dst, long long b, int o, long long n, const float (&v)[4]) {
    if constexpr (TYPE == 0) {
        float* d = static_cast<float*>(dst) + b;
        if constexpr (VEC) {
            put<NT>(d + o, f32x4_4{v[0], v[1], v[2], v[3]});
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (b + o + e < n) d[o + e] = v[e];
        }
    } else {
        uint16_t* d = static_cast<uint16_t*>(dst) + b;
        if constexpr (VEC) {
            using H = std::conditional_t<TYPE == 1, __bf16, _Float16>;
            typedef H h2 __attribute__((ext_vector_type(2)));
            put<NT>(d + o, u32x2_2{__builtin_bit_cast(uint32_t, h2{(H)v[0], (H)v[1]}), __builtin_bit_cast(uint32_t, h2{(H)v[2], (H)v[3]})});
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (b + o + e < n) d[o + e] = to16(v[e], TYPE);
        }
    }
}
template <bool VEC, bool NT>
__device__ __forceinline__ uint32_t load_codes(const void* src, long long b, int o, long long n) {
    const uint8_t* s = static_cast<const uint8_t*>(src) + b;
    if constexpr (VEC) return get<NT>(s + o);
    uint32_t u = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (b + o + e < n) u |= (uint32_t)s[o + e] << (8 * e);
    return u;
}
template <bool VEC, bool NT>
__device__ __forceinline__ void store_codes(void* dst, long long b, int o, long long n, uint32_t u) {
    uint8_t* d = static_cast<uint8_t*>(dst) + b;
    if constexpr (VEC) {
        put<NT>(d + o, u);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (b + o + e < n) d[o + e] = (uint8_t)(u >> (8 * e));
    }
}

// 2^e for e in [-126, 127]
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }
__device__ __forceinline__ bool finite(float x) { return (__builtin_bit_cast(uint32_t, x) & 0x7f800000u) != 0x7f800000u; }

// e4m3 code of y in [0, 256), u in [0, 2^16): the low 20 bits of the fp32 pattern are the part of a step that is decided by
// the random bits.  Below the smallest normal code the steps are even: adding 2^-6 there gives the pattern the same form.
__device__ __forceinline__ uint32_t encode(float y, uint32_t u) {
    const bool small = y < 0x1p-6f;
    const uint32_t bits = __builtin_bit_cast(uint32_t, small ? y + 0x1p-6f : y), zero = (small ? 0u - (968u << 20) : 0u - (960u << 20)) + 8u;
    return (bits + (u << 4) + zero) >> 20;
}

struct AwStep {
    float size, keep, b1, c1, b2, c2, eps, gs, inv2;
};
// Square root rounded to the nearest.  The hardware's is within one unit of it, and Tuckerman's test says which of s and the two
// values next to it is nearest: r is, where r (r - u) < x <= r (r + u), u one unit.
__device__ __forceinline__ float root_of(float x) {
    const float s = __builtin_amdgcn_sqrtf(x);
    const float lo = __builtin_bit_cast(float, __builtin_bit_cast(int, s) - 1), hi = __builtin_bit_cast(float, __builtin_bit_cast(int, s) + 1);
    float r = __builtin_fmaf(-lo, s, x) <= 0.f ? lo : s;
    r = __builtin_fmaf(-hi, s, x) > 0.f ? hi : r;
    return r;           // s itself for zero, infinity and NaN: one of s' is no number there, and no comparison holds
}
// The hardware takes denormals for zero, and the test's differences are lost among them: where a lane of the wave holds a v below
// 2^-64, the roots are taken of 2^64 v.  (Scaling in every case: 46 M elements in bf16 with 8-bit states 95.0 -> 98.6 us.)
__device__ __forceinline__ void roots(const float (&v)[4], float (&r)[4]) {
    const bool tiny = __builtin_fminf(__builtin_fminf(v[0], v[1]), __builtin_fminf(v[2], v[3])) < 0x1p-64f;
    if (__builtin_amdgcn_ballot_w64(tiny) == 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = root_of(v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool up = v[e] < 0x1p-64f;
            r[e] = root_of(v[e] * (up ? 0x1p64f : 1.f)) * (up ? 0x1p-32f : 1.f);
        }
    }
}
// p is rounded to its own type once more than anything here errs: the quotient is a product with the hardware's reciprocal
// (one unit off at most).
__device__ __forceinline__ void update(const AwStep& s, float (&p)[4], const float (&g)[4], float (&m)[4], float (&v)[4], float (&root)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float x = g[e] * s.gs;
        m[e] = m[e] * s.b1 + x * s.c1;
        v[e] = v[e] * s.b2 + (x * x) * s.c2;
    }
    roots(v, root);
#pragma unroll
    for (int e = 0; e < 4; ++e) p[e] = __builtin_fmaf(-(m[e] * s.size), __builtin_amdgcn_rcpf(__builtin_fmaf(root[e], s.inv2, s.eps)), p[e] * s.keep);
}

template <int PT, int GT, bool VEC, bool NT>
__device__ __forceinline__ void body32(const AwTensor& t, const AwStep& s, long long b, int o) {
    float p[4], g[4], m[4], v[4], root[4];
    load4<PT, VEC, NT>(t.p, b, o, t.n, p);
    load4<GT, VEC, NT>(t.g, b, o, t.n, g);
    load4<0, VEC, NT>(t.m, b, o, t.n, m);
    load4<0, VEC, NT>(t.v, b, o, t.n, v);
    update(s, p, g, m, v, root);
    store4<PT, VEC, NT>(t.p, b, o, t.n, p);
    store4<0, VEC, NT>(t.m, b, o, t.n, m);
    store4<0, VEC, NT>(t.v, b, o, t.n, v);
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    const auto step = [](uint32_t v, uint32_t o) { return max(v, o); };
    v = step(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));
    v = step(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));
    v = step(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));
    v = step(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true));
    v = step(v, (uint32_t)__shfl_xor((int)v, 16, 64));
    return step(v, (uint32_t)__shfl_xor((int)v, 32, 64));
}

// one block of 256 elements by one wave, four elements a lane from i on
template <int PT, int GT, bool VEC, bool NT>
struct Block8 {
    float p[4], g[4], ms, rs;
    uint32_t cm, cv;
    __device__ __forceinline__ void load(const AwTensor& t, long long i, int o) {
        load4<PT, VEC, NT>(t.p, i, o, t.n, p);
        load4<GT, VEC, NT>(t.g, i, o, t.n, g);
        cm = load_codes<VEC, NT>(t.m, i, o, t.n);
        cv = load_codes<VEC, NT>(t.v, i, o, t.n);
        ms = t.ms[i / AW_BLOCK];
        rs = t.rs[i / AW_BLOCK];
    }
    __device__ __forceinline__ void step(const AwTensor& t, const AwStep& s, long long i, int o, uint32_t key) {
        float m[4], v[4], r[4];
        m[0] = __builtin_amdgcn_cvt_f32_fp8(cm, 0) * ms;
        m[1] = __builtin_amdgcn_cvt_f32_fp8(cm, 1) * ms;
        m[2] = __builtin_amdgcn_cvt_f32_fp8(cm, 2) * ms;
        m[3] = __builtin_amdgcn_cvt_f32_fp8(cm, 3) * ms;
        v[0] = __builtin_amdgcn_cvt_f32_fp8(cv, 0) * rs;
        v[1] = __builtin_amdgcn_cvt_f32_fp8(cv, 1) * rs;
        v[2] = __builtin_amdgcn_cvt_f32_fp8(cv, 2) * rs;
        v[3] = __builtin_amdgcn_cvt_f32_fp8(cv, 3) * rs;
        // magnitudes are compared as patterns: infinities and NaN come out on top, and only then are they looked for
        uint32_t mmax = 0, vmax = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = v[e] * v[e];
        update(s, p, g, m, v, r);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            mmax = max(mmax, __builtin_bit_cast(uint32_t, m[e]) & 0x7fffffffu);
            vmax = max(vmax, __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu);
        }
        store4<PT, VEC, NT>(t.p, i, o, t.n, p);
        mmax = wave_max(mmax);
        vmax = wave_max(vmax);
        const bool odd = __builtin_amdgcn_readfirstlane(max(mmax, vmax)) >= 0x7f800000;
        uint32_t no_m = 0, no_v = 0;        // codes of what is not finite, which counts as zero in what follows
        if (odd) {
            mmax = vmax = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (!finite(m[e])) {
                    no_m |= 0x7fu << (8 * e);
                    m[e] = __builtin_copysignf(0.f, m[e]);
                }
                if (!finite(v[e])) {
                    no_v |= 0x7fu << (8 * e);
                    v[e] = r[e] = 0.f;
                }
                mmax = max(mmax, __builtin_bit_cast(uint32_t, m[e]) & 0x7fffffffu);
                vmax = max(vmax, __builtin_bit_cast(uint32_t, v[e]));
            }
            mmax = wave_max(mmax);
            vmax = wave_max(vmax);
        }
        const int em = max((int)(mmax >> 23) - 127, -100) - 7, er = (max((int)(vmax >> 23) - 127, -126) >> 1) - 7;
        const float im = pow2(-em), ir = pow2(-er);
        uint32_t nm = no_m, nr = no_v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t h = mix(key ^ ((uint32_t)i + (uint32_t)(o + e)));
            const uint32_t a = encode(__builtin_fabsf(m[e]) * im, h & 0xffffu);
            const uint32_t b = max(encode(r[e] * ir, h >> 16), min(__builtin_bit_cast(uint32_t, v[e]), 1u));
            nm |= (a | ((__builtin_bit_cast(uint32_t, m[e]) >> 24) & 0x80u)) << (8 * e);
            nr |= b << (8 * e);
        }
        store_codes<VEC, NT>(t.m, i, o, t.n, nm);
        store_codes<VEC, NT>(t.v, i, o, t.n, nr);
        if ((threadIdx.x & 63) == 0) {
            t.ms[i / AW_BLOCK] = pow2(em);
            t.rs[i / AW_BLOCK] = pow2(er);
        }
    }
};

template <int BITS, bool NT, int PT, int GT>
__device__ __forceinline__ void chunk(const AwTensor& t, const AwStep& s, long long at, uint32_t key) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if constexpr (BITS == 32) {
#pragma unroll
        for (int u = 0; u < AW_CHUNK / 1024; ++u) {
            const long long b = at + u * 1024 + wave * 256;
            if (b + 256 <= t.n) {
                body32<PT, GT, true, NT>(t, s, b, lane * 4);
            } else if (b + lane * 4 < t.n) {
                body32<PT, GT, false, NT>(t, s, b, lane * 4);
            }
        }
    } else {
        // two blocks of 256 a wave, the second one's reads under way while the first is computed
        const long long b = at + wave * (2 * AW_BLOCK);
        if (b + 2 * AW_BLOCK <= t.n) {
            Block8<PT, GT, true, NT> x, y;
            x.load(t, b, lane * 4);
            y.load(t, b + AW_BLOCK, lane * 4);
            x.step(t, s, b, lane * 4, key);
            y.step(t, s, b + AW_BLOCK, lane * 4, key);
        } else {
            for (int u = 0; u < 2; ++u) {
                const long long i = b + u * AW_BLOCK;
                if (i >= t.n) break;
                Block8<PT, GT, false, NT> x;
                x.load(t, i, lane * 4);
                x.step(t, s, i, lane * 4, key);
            }
        }
    }
}

template <int BITS, bool NT>
__global__ __launch_bounds__(256) void adamw_kernel(const AwArgs a) {
    // the block's tensor: the lanes compare it with every tensor's first chunk at once
    const int lane = threadIdx.x & 63;
    const unsigned first = lane < a.n ? a.first[lane] : 0xffffffffu;
    const int k = __builtin_popcountll(__ballot(first <= blockIdx.x)) - 1;
    const AwTensor& t = a.t[k];
    const long long at = (long long)(blockIdx.x - a.first[k]) * AW_CHUNK;
    AwStep s{t.size, t.keep, a.b1, a.c1, a.b2, a.c2, a.eps, a.gs, a.inv2};
    uint32_t step = (uint32_t)a.step;
    if (a.step_dev) {
        step = (uint32_t)a.step_dev[0];
        s.size = t.size * __builtin_bit_cast(float, a.step_dev[1]);
        s.inv2 = __builtin_bit_cast(float, a.step_dev[2]);
    }
    const uint32_t key = BITS == 8 ? mix(a.seed + step * 0xA54FF53Bu + (uint32_t)t.index * 0x3C6EF373u) : 0u;
    switch (t.types) {
        case 0: chunk<BITS, NT, 0, 0>(t, s, at, key); break;
        case 1: chunk<BITS, NT, 1, 0>(t, s, at, key); break;
        case 2: chunk<BITS, NT, 2, 0>(t, s, at, key); break;
        case 3: chunk<BITS, NT, 0, 1>(t, s, at, key); break;
        case 4: chunk<BITS, NT, 1, 1>(t, s, at, key); break;
        case 5: chunk<BITS, NT, 2, 1>(t, s, at, key); break;
        case 6: chunk<BITS, NT, 0, 2>(t, s, at, key); break;
        case 7: chunk<BITS, NT, 1, 2>(t, s, at, key); break;
        default: chunk<BITS, NT, 2, 2>(t, s, at, key); break;
    }
}

// counter[0] += 1; counter[1], [2] = 1 / (1 - b1^t), 1 / sqrt(1 - b2^t) as fp32 patterns
__global__ void adamw_tick_kernel(int* counter, double b1, double b2) {
    const int t = counter[0] + 1;
    counter[0] = t;
    counter[1] = __builtin_bit_cast(int, (float)(1.0 / (1.0 - pow(b1, (double)t))));
    counter[2] = __builtin_bit_cast(int, (float)(1.0 / sqrt(1.0 - pow(b2, (double)t))));
}

inline bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

struct Span {
    uintptr_t lo, hi;
};

}  // namespace

extern "C" {

int pgan_adamw_multi(void* const* p, const void* const* g, void* const* m, void* const* v, float* const* m_scale,
                     float* const* r_scale, const long long* numel, const int* types, const double* lr,
                     const double* decay, int n, int bits, double b1, double b2, float eps, float grad_scale, int seed,
                     int* step_dev, int step, hipStream_t st) {
    if (n < 0 || (bits != 32 && bits != 8) || !(b1 >= 0 && b1 < 1) || !(b2 >= 0 && b2 < 1)) return PGAN_EINVAL;
    if (!(eps == 0 || eps >= 0x1p-126f)) return PGAN_EINVAL;     // the hardware's reciprocal takes denormals for zero
    if (!step_dev && step < 1) return PGAN_EINVAL;
    if (n > 0 && (!p || !g || !m || !v || !numel || !types || !lr || !decay)) return PGAN_EINVAL;
    if (bits == 8 && n > 0 && (!m_scale || !r_scale)) return PGAN_EINVAL;
    const int size_of[3] = {4, 2, 2};
    long long bytes = 0;
    try {
        // what is written: no two of these may share memory (the same tensor twice in the lists, a state for two of them)
        std::vector<Span> out, in;
        out.reserve((size_t)n * 5 + 1);
        in.reserve((size_t)n);
        const auto add = [](std::vector<Span>& to, const void* q, long long bytes) {
            const uintptr_t lo = reinterpret_cast<uintptr_t>(q);
            to.push_back(Span{lo, lo + (uintptr_t)bytes});
        };
        for (int i = 0; i < n; ++i) {
            if (numel[i] < 0 || numel[i] > AW_MOST * AW_CHUNK || types[i] < 0 || types[i] > 8) return PGAN_EINVAL;
            if (numel[i] == 0) continue;
            if (!p[i] || !g[i] || !m[i] || !v[i] || (bits == 8 && (!m_scale[i] || !r_scale[i]))) return PGAN_EINVAL;
            const int ps = size_of[types[i] % 3], gsz = size_of[types[i] / 3];
            if (!aligned(p[i], ps) || !aligned(g[i], gsz)) return PGAN_EINVAL;
            if (bits == 32 && (!aligned(m[i], 4) || !aligned(v[i], 4))) return PGAN_EINVAL;
            bytes += numel[i] * (2 * ps + gsz + bits / 2);
            add(in, g[i], numel[i] * gsz);
            add(out, p[i], numel[i] * ps);
            add(out, m[i], numel[i] * (bits / 8));
            add(out, v[i], numel[i] * (bits / 8));
            if (bits == 8) {
                const long long nb = (numel[i] + AW_BLOCK - 1) / AW_BLOCK * 4;
                add(out, m_scale[i], nb);
                add(out, r_scale[i], nb);
            }
        }
        if (step_dev) add(out, step_dev, 16);
        std::sort(out.begin(), out.end(), [](const Span& x, const Span& y) { return x.lo < y.lo; });
        for (size_t i = 1; i < out.size(); ++i)
            if (out[i].lo < out[i - 1].hi) return PGAN_EINVAL;
        // nor may a gradient with any of them
        for (const Span& s : in) {
            const auto next = std::partition_point(out.begin(), out.end(), [&s](const Span& o) { return o.hi <= s.lo; });
            if (next != out.end() && next->lo < s.hi) return PGAN_EINVAL;
        }
    } catch (...) {
        return PGAN_EINVAL;
    }
    // Steps of more than one and a half times the memory-side cache go past the caches: what passes between two steps leaves
    // little of them there.  us with ordinary accesses and past the caches, after 1 GB of other writes: 240 MB 58 and 46 (fp32,
    // 32 bits), 63 and 46 (fp32, 8), 64 and 54 (bf16, 8); 450 MB 102 and 81, 105 and 79, 107 and 92; step after step with
    // nothing between: 240 MB 37 and 41, 40 and 42, 49 and 50; 450 MB 67 and 77, 72 and 76, 94 and 90; 1200 MB 232 and 218, 222
    // and 192, 246 and 241.  Smaller steps do not: an iteration of the trainer (78 MB a step, the weights read again at once)
    // takes 6.17 ms and 6.18.
    const bool past = bytes > (384LL << 20);
    if (step_dev) adamw_tick_kernel<<<1, 1, 0, st>>>(step_dev, b1, b2);
    AwArgs a;
    a.step_dev = step_dev;
    a.step = step;
    a.b1 = (float)b1;
    a.c1 = (float)(1.0 - b1);
    a.b2 = (float)b2;
    a.c2 = (float)(1.0 - b2);
    a.eps = eps;
    a.gs = grad_scale;
    a.seed = (unsigned)seed;
    const double bc1 = step_dev ? 1.0 : 1.0 - pow(b1, (double)step);
    a.inv2 = step_dev ? 1.f : (float)(1.0 / sqrt(1.0 - pow(b2, (double)step)));
    int i = 0;
    while (i < n) {
        a.n = 0;
        long long chunks = 0;
        for (; i < n && a.n < AW_MAX; ++i) {
            if (numel[i] == 0) continue;
            const long long c = (numel[i] + AW_CHUNK - 1) / AW_CHUNK;
            if (chunks + c > AW_MOST) break;
            a.first[a.n] = (unsigned)chunks;
            a.t[a.n] = AwTensor{p[i], g[i], m[i], v[i], bits == 8 ? m_scale[i] : nullptr, bits == 8 ? r_scale[i] : nullptr,
                                numel[i], (float)(lr[i] / bc1), (float)(1.0 - lr[i] * decay[i]), types[i], i};
            chunks += c;
            ++a.n;
        }
        if (a.n == 0) break;
        auto* const kernel = bits == 32 ? (past ? adamw_kernel<32, true> : adamw_kernel<32, false>) : past ? adamw_kernel<8, true> : adamw_kernel<8, false>;
        kernel<<<(unsigned)chunks, 256, 0, st>>>(a);
    }
    return pgan_launch_status();
}

}  // extern "C"
