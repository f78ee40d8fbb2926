// The 4-bit cache is written and read back (layout: cache4.cuh).  Both directions move bytes: of a bf16 row of 128 columns 256 bytes
// on the dense side and 80 in the cache.  A thread takes eight neighbouring columns of four positions (a multiple of four and the next
// three): those are one word of each key row or two 8-byte words of a value tile, four threads are a group, and threads run along rows.
// Four rows a thread keep enough loads in flight, and values leave in pieces of 8 bytes instead of 2.  Measured, 163840 rows of 128 columns
// (2 x 8 x 2048 x 5): written from bf16 in 19.0 us (2.9 TB/s; latency: 19 instructions a column fill 0.6 of the issue slots, and
// the warps that 48 registers leave room for not the rest: with the columns as float32 in 62 registers 26, with eight rows a thread in 64
// registers 26.7), from float32 in 18.6 (5.2 TB/s); read as bf16 in 9.6 us (5.7 TB/s), as float32 in 15.2 (6.4).
#include <type_traits>

#include "cache4.cuh"

namespace rb {

constexpr int C4_THREADS = 128;

// Where eight columns (c8 of a row) of positions quad .. quad + 3 lie.  Keys: a word, `next` bytes to the next position; values: four 16-bit
// words in a row, and `next` bytes behind them those of the next part g.  group: s and m of the first position, group_next to the next.
struct Place {
    unsigned char* codes;
    size_t group;
    int next, group_next;
    __device__ __forceinline__ Place(const Cache4View& c, int part, int b, uint32_t h, int quad, uint32_t c8) {
        const int NG = c.dim / C4_GROUP, j = c8 >> 2, t = c8 & 3;
        const size_t head = ((size_t)b * c.kv_heads + h) * c.max_seq;
        if (part == 0) {
            codes = c.codes[0] + (head + quad) * (NG * 16) + (t * NG + j) * 4;
            next = NG * 16;
            group = (head + quad) * NG + j;
            group_next = NG;
        } else {
            codes = c.codes[1] + (head + (quad & ~15)) * (NG * 16) + 2 * value_at(NG, j, 2 * t, quad & 15);
            next = 2 * (value_at(NG, j, 1, 0) - value_at(NG, j, 0, 0));
            group = (head + quad) * NG + j * 4;
            group_next = 1;
        }
    }
};

struct Cache4Store {
    Cache4View c;
    const void* src[2];
    size_t sb[2], ss[2], sh[2];  // strides of sequence, position and head, in elements
    bool wide[2];                // rows begin at multiples of 16 bytes
    Past past;
    int seq;
    uint32_t units;              // quads * kv_heads * dim / 8
    FastDiv per_row, heads;
};

// s of a group.  The definition rounds the quotient in 64 bits to float32 and then to float16.  float32 arithmetic gives the same
// float16 unless its result is within a few of its own steps of a border between two float16 numbers.
__device__ __forceinline__ __half group_step(float low, float high) {
    const float q = (high - low) * (1.f / 15.f);
    const int low_bits = __float_as_int(q) & 0x1fff;  // of a normal float16 these are cut off, and 0x1000 is the border
    if (high > low && (q < 6.2e-5f || (low_bits >= 0x1000 - 4 && low_bits <= 0x1000 + 4)))
        return __float2half_rn((float)(((double)high - (double)low) / 15.0));
    return __float2half_rn(q);
}

__device__ __forceinline__ float fast_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Eight neighbouring columns as they came: 16-bit ones stay two in a word until they are needed (half the registers, and a minimum of two is
// one instruction).
template <typename T>
struct Eight {
    uint32_t w[4];
    using Two = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    __device__ __forceinline__ Two two(int n) const { return *reinterpret_cast<const Two*>(&w[n]); }
    __device__ __forceinline__ void none() { w[0] = w[1] = w[2] = w[3] = 0u; }
    __device__ __forceinline__ void load(const T* p, bool wide) {
        if (wide) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
            for (int n = 0; n < 4; ++n) w[n] = h[2 * n] | (uint32_t)h[2 * n + 1] << 16;
        }
    }
    // (minimum and maximum pass over NaN)
    __device__ __forceinline__ void bounds(float& lo, float& hi) const {
        const Two a = __hmin2(__hmin2(two(0), two(1)), __hmin2(two(2), two(3))), b = __hmax2(__hmax2(two(0), two(1)), __hmax2(two(2), two(3)));
        lo = fminf(type_load(&a.x), type_load(&a.y));
        hi = fmaxf(type_load(&b.x), type_load(&b.y));
    }
    __device__ __forceinline__ float2 pair(int n) const {
        const Two a = two(n);
        return make_float2(type_load(&a.x), type_load(&a.y));
    }
};
template <>
struct Eight<float> {
    float x[8];
    __device__ __forceinline__ void none() {
#pragma unroll
        for (int n = 0; n < 8; ++n) x[n] = 0.f;
    }
    __device__ __forceinline__ void load(const float* p, bool wide) {
        if (wide) {
            const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
#pragma unroll
            for (int n = 0; n < 8; ++n) x[n] = p[n];
        }
    }
    __device__ __forceinline__ void bounds(float& lo, float& hi) const {
        lo = hi = x[0];
#pragma unroll
        for (int n = 1; n < 8; ++n) {
            lo = fminf(lo, x[n]);
            hi = fmaxf(hi, x[n]);
        }
    }
    __device__ __forceinline__ float2 pair(int n) const { return make_float2(x[2 * n], x[2 * n + 1]); }
};

// Smallest and largest of the groups of four rows x[k], of which each of four neighbouring threads holds eight columns: thread t of the
// four gets those of row t.  (Rows are handed over by halves, so that every thread makes one row's s and m and not all four.)
template <typename T>
__device__ __forceinline__ void group_bounds(const Eight<T> (&x)[4], int t, float& low, float& high) {
    float lo[4], hi[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k].bounds(lo[k], hi[k]);
    const bool up = t & 2, odd = t & 1;
    float l[2], h[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        l[k] = fminf(up ? lo[k + 2] : lo[k], __shfl_xor_sync(0xffffffffu, up ? lo[k] : lo[k + 2], 2));
        h[k] = fmaxf(up ? hi[k + 2] : hi[k], __shfl_xor_sync(0xffffffffu, up ? hi[k] : hi[k + 2], 2));
    }
    low = fminf(odd ? l[1] : l[0], __shfl_xor_sync(0xffffffffu, odd ? l[0] : l[1], 1));
    high = fmaxf(odd ? h[1] : h[0], __shfl_xor_sync(0xffffffffu, odd ? h[0] : h[1], 1));
}

// s (low half) and m of a group.  A group of nothing but NaN holds zeros.  s is never negative: its sign marks a float32 group with columns
// above 65504, which are quantised as that.
constexpr uint32_t C4_BEYOND = 0x8000u;
template <typename T>
__device__ __forceinline__ uint32_t group_params(float low, float high) {
    if (low != low) low = high = 0.f;
    const uint32_t beyond = sizeof(T) == 4 && high > C4_MOST ? C4_BEYOND : 0u;
    low = fminf(fmaxf(low, -C4_MOST), C4_MOST);
    high = fminf(fmaxf(high, -C4_MOST), C4_MOST);
    return (uint32_t)__half_as_ushort(group_step(low, high)) | beyond | (uint32_t)__half_as_ushort(__float2half_rn(low)) << 16;
}

// The codes of eight columns, column n in bits 4 n.
template <typename T>
__device__ __forceinline__ uint32_t quantise8(Eight<T> x, uint32_t params) {
    if constexpr (sizeof(T) == 4) {
        // Where m is rounded up to 65504 or near it, 65504 is not the highest code, which larger columns would get.  (m of 16-bit types
        // is not rounded and s by 2^-11 at most: 65504 is within a hundredth of the highest code.)
        if (params & C4_BEYOND) {
#pragma unroll
            for (int n = 0; n < 8; ++n) x.x[n] = x.x[n] > C4_MOST ? C4_MOST : x.x[n];  // (NaN stays)
            params &= ~C4_BEYOND;
        }
    }
    const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(&params));
    const float s = sm.x, m = sm.y, inv = s > 0.f ? fast_rcp(s) : 0.f, inv15 = inv * (1.f / 15.f);
    // the quotient over 15, kept within 0 .. 1 (NaN: 0); 1.5 2^23 + 15 times that is a whole number, to the nearest, ties to even
    constexpr float round_at = 12582912.f;
    const float2 minus_m = make_float2(-m, -m), fifteen = make_float2(15.f, 15.f), to_whole = make_float2(round_at, round_at),
                 back = make_float2(-round_at, -round_at), minus = make_float2(-1.f, -1.f);
    float2 code[4];
    float off = 0.f;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const float2 d = __fadd2_rn(x.pair(n), minus_m);
        const float2 q = make_float2(__saturatef(d.x * inv15), __saturatef(d.y * inv15));
        code[n] = __fadd2_rn(__ffma2_rn(q, fifteen, to_whole), back);
        const float2 e = __ffma2_rn(code[n], minus, __fmul2_rn(q, fifteen));
        off = fmaxf(off, fmaxf(fabsf(e.x), fabsf(e.y)));
    }
    // The quotient in float32 is off by less than 1e-5: of what lies that near to a border k + 1/2 between two codes, x - m is compared with
    // (k + 1/2) s exactly: that is a product of 11 and 5 bits, x - m is the sum of its rounded value and of what the rounding left, and the
    // difference of two numbers that near to one another is exact.  (Types of few bits come here often: (x - m) / s is a ratio of small
    // numbers, and of 256 bf16 columns one lies on a border in a seventh of the cases.)
    if (off > 0.5f - 2e-5f) {
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            float& c = n & 1 ? code[n >> 1].y : code[n >> 1].x;
            const float2 two = x.pair(n >> 1);
            const float value = n & 1 ? two.y : two.x, q = fminf(fmaxf((value - m) * inv, 0.f), 15.f);
            if (fabsf(q - c) > 0.5f - 4e-5f) {
                const float below = floorf(q);
                const float t = value - m, taken = t - value, left = (value - (t - taken)) - (m + taken);
                const float d = (t - (below + 0.5f) * s) + left;
                c = below + (d > 0.f || (d == 0.f && ((int)below & 1)) ? 1.f : 0.f);
            }
        }
    }
    // (four codes are a number below 2^16, which the sum with 2^23 has in its low bits)
    uint32_t half[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float2 c0 = code[2 * k], c1 = code[2 * k + 1];
        half[k] = __float_as_uint(fmaf(fmaf(fmaf(c1.y, 16.f, c1.x), 16.f, c0.y), 16.f, c0.x) + 8388608.f);
    }
    return __byte_perm(half[0], half[1], 0x5410);
}

template <typename T>
__global__ void __launch_bounds__(C4_THREADS, sizeof(T) == 4 ? 8 : 10) cache4_store_kernel(const __grid_constant__ Cache4Store p) {
    pdl_wait();
    pdl_trigger();
    const uint32_t u = blockIdx.x * C4_THREADS + threadIdx.x;
    const int b = blockIdx.y, part = blockIdx.z;
    const bool on = u < p.units;
    const uint32_t row = p.per_row.div(on ? u : 0), c8 = (on ? u : 0) - row * p.per_row.d;
    const uint32_t nth = p.heads.div(row), h = row - nth * p.heads.d;
    const int past = past_of(p.past, b), quad = (past & ~3) + 4 * (int)nth;
    const int from = max(past - quad, 0), to = min(min(past + p.seq, p.c.max_seq) - quad, 4);  // which of the four are there
    const T* src = static_cast<const T*>(p.src[part]) + (size_t)b * p.sb[part] + (size_t)h * p.sh[part] + c8 * 8;
    Eight<T> x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (k >= from && k < to) x[k].load(src + (size_t)(quad + k - past) * p.ss[part], p.wide[part]);
        else x[k].none();
    }
    float low, high;
    group_bounds(x, c8 & 3, low, high);
    const uint32_t own = group_params<T>(low, high);
    uint32_t word[4];
    __half s[4], m[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t params = __shfl_sync(0xffffffffu, own, (threadIdx.x & 28) + k);
        word[k] = quantise8(x[k], params);
        s[k] = __ushort_as_half((unsigned short)(params & ~C4_BEYOND));
        m[k] = __ushort_as_half((unsigned short)(params >> 16));
    }
    if (!on || from >= to) return;
    const Place w(p.c, part, b, h, quad, c8);
    const bool whole = from == 0 && to == 4, first = (c8 & 3) == 0;
    __half *step = p.c.step[part] + w.group, *least = p.c.least[part] + w.group;
    if (part == 0) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (k >= from && k < to) {
                *reinterpret_cast<uint32_t*>(w.codes + k * w.next) = word[k];
                if (first) step[k * w.group_next] = s[k], least[k * w.group_next] = m[k];
            }
        }
    } else if (whole) {
        *reinterpret_cast<uint2*>(w.codes) = make_uint2(__byte_perm(word[0], word[1], 0x5410), __byte_perm(word[2], word[3], 0x5410));
        *reinterpret_cast<uint2*>(w.codes + w.next) = make_uint2(__byte_perm(word[0], word[1], 0x7632), __byte_perm(word[2], word[3], 0x7632));
        if (first) {
            auto two = [](__half a, __half c) { return (uint32_t)__half_as_ushort(a) | (uint32_t)__half_as_ushort(c) << 16; };
            *reinterpret_cast<uint2*>(step) = make_uint2(two(s[0], s[1]), two(s[2], s[3]));
            *reinterpret_cast<uint2*>(least) = make_uint2(two(m[0], m[1]), two(m[2], m[3]));
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (k >= from && k < to) {
                reinterpret_cast<uint16_t*>(w.codes)[k] = (uint16_t)word[k];
                reinterpret_cast<uint16_t*>(w.codes + w.next)[k] = (uint16_t)(word[k] >> 16);
                if (first) step[k] = s[k], least[k] = m[k];
            }
        }
    }
}

struct Cache4Load {
    Cache4View c;
    void* dst[2];
    int begin, span;
    bool whole;      // float32 rows begin at multiples of 32 bytes
    uint32_t units;  // kv_heads * quads * dim / 8
    FastDiv per_row, quads;
    // rows for a prompt
    int seq, window, negate;
    Past past;
    int* past_out;
};

// 32 bytes at once, at a multiple of that: two stores of 16 reach L2 as two halves of every sector (22.8 us instead of 15.2 for 97 MB).
__device__ __forceinline__ void store8_whole(float* p, const float (&x)[8]) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]),
                 "f"(x[5]), "f"(x[6]), "f"(x[7])
                 : "memory");
}

template <typename T, bool PROMPT>
__global__ void __launch_bounds__(C4_THREADS) cache4_load_kernel(const __grid_constant__ Cache4Load p) {
    pdl_wait();
    pdl_trigger();
    const uint32_t u = blockIdx.x * C4_THREADS + threadIdx.x;
    const int b = blockIdx.y, part = blockIdx.z;
    if (u >= p.units) return;
    const uint32_t row = p.per_row.div(u), c8 = u - row * p.per_row.d;
    const uint32_t h = p.quads.div(row);
    const int quad = (p.begin & ~3) + 4 * (int)(row - h * p.quads.d), end = p.begin + p.span;
    int limit = p.c.max_seq;  // positions from here on are zeros
    if constexpr (PROMPT) {
        // the attention reads tiles of 128 positions from the first one its first query sees: a head's rows end in zeros, and so begin
        // the rows that a tile at the end of the head before reaches into
        const int past = past_of(p.past, b);
        limit = min(past + p.seq, p.c.max_seq);
        if (p.past_out && u == 0 && part == 0) p.past_out[b] = past;
        if (quad >= limit + 128 || (quad + 3 < first_visible(past, 0, p.window) && quad >= 128)) return;
    }
    uint32_t word[4] = {0u, 0u, 0u, 0u};
    float s[4] = {0.f, 0.f, 0.f, 0.f}, m[4] = {0.f, 0.f, 0.f, 0.f};
    if (quad < p.c.max_seq) {
        const Place w(p.c, part, b, h, quad, c8);
        const __half *step = p.c.step[part] + w.group, *least = p.c.least[part] + w.group;
        if (part == 0) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                word[k] = *reinterpret_cast<const uint32_t*>(w.codes + k * w.next);
                s[k] = __half2float(step[k * w.group_next]);
                m[k] = __half2float(least[k * w.group_next]);
            }
        } else {
            const uint2 lo = *reinterpret_cast<const uint2*>(w.codes), hi = *reinterpret_cast<const uint2*>(w.codes + w.next);
            const uint2 sv = *reinterpret_cast<const uint2*>(step), mv = *reinterpret_cast<const uint2*>(least);
            word[0] = __byte_perm(lo.x, hi.x, 0x5410), word[1] = __byte_perm(lo.x, hi.x, 0x7632);
            word[2] = __byte_perm(lo.y, hi.y, 0x5410), word[3] = __byte_perm(lo.y, hi.y, 0x7632);
            const uint32_t sw[2] = {sv.x, sv.y}, mw[2] = {mv.x, mv.y};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&sw[k >> 1])), c = __half22float2(*reinterpret_cast<const __half2*>(&mw[k >> 1]));
                s[k] = k & 1 ? a.y : a.x;
                m[k] = k & 1 ? c.y : c.x;
            }
        }
    }
    const bool negate = PROMPT && part == 0 && p.negate;
    T* dst = static_cast<T*>(p.dst[part]) + (((size_t)b * p.c.kv_heads + h) * p.span) * p.c.dim + c8 * 8;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int pos = quad + k;
        if (pos < p.begin || pos >= end) continue;
        if (PROMPT && pos >= limit) s[k] = m[k] = 0.f;
        if (negate) s[k] = -s[k], m[k] = -m[k];
        // The sum of 2^23 and a code where it stands in its half of the word is a matter of bits, and that difference times s over the power
        // of 16 is s code (conversions from integers take 16 a clock, which bounded the kernel).
        const float s16 = s[k] * 0.0625f;
        const float2 m2 = make_float2(m[k], m[k]), back = make_float2(-8388608.f, -8388608.f), step2[2] = {make_float2(s[k], s16),
            make_float2(s16 * 0.0625f, s16 * 0.00390625f)};
        float x[8];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const uint32_t half = n < 2 ? word[k] : word[k] >> 16;
            const int at = n & 1 ? 8 : 0;
            const float2 c = make_float2(__uint_as_float((half & (15u << at)) | 0x4b000000u), __uint_as_float((half & (240u << at)) | 0x4b000000u));
            float2 y = __ffma2_rn(__fadd2_rn(c, back), step2[n & 1], m2);
            if (std::is_same<T, __half>::value)  // (m + 15 s may lie a rounding above the largest float16)
                y = make_float2(fminf(fmaxf(y.x, -C4_MOST), C4_MOST), fminf(fmaxf(y.y, -C4_MOST), C4_MOST));
            x[2 * n] = y.x;
            x[2 * n + 1] = y.y;
        }
        T* to = dst + (size_t)(pos - p.begin) * p.c.dim;
        if constexpr (sizeof(T) == 4) {
            if (p.whole) {
                store8_whole(to, x);
                continue;
            }
        }
        store8(to, x);
    }
}

int cache4_view(const rotor_b200_cache4* c, Cache4View& v) {
    RB_REQUIRE(c && c->batch > 0 && c->kv_heads > 0 && c->max_seq > 0 && c->k_codes && c->v_codes && c->k_step && c->k_least && c->v_step &&
               c->v_least);
    const uintptr_t all = (uintptr_t)c->k_codes | (uintptr_t)c->v_codes | (uintptr_t)c->k_step | (uintptr_t)c->k_least |
                          (uintptr_t)c->v_step | (uintptr_t)c->v_least;
    RB_REQUIRE((all & 15) == 0);
    const int g = c->dim / C4_GROUP;
    if (c->dim % C4_GROUP || !(g >= 1 && (g <= 4 || g == 6 || g == 8)) || c->max_seq % C4_POSITIONS || c->batch > 65535 || c->kv_heads > 65535 ||
        c->max_seq > (1 << 26))
        return ROTOR_B200_ERR_SHAPE;
    v.codes[0] = c->k_codes;
    v.codes[1] = c->v_codes;
    v.step[0] = static_cast<__half*>(c->k_step);
    v.step[1] = static_cast<__half*>(c->v_step);
    v.least[0] = static_cast<__half*>(c->k_least);
    v.least[1] = static_cast<__half*>(c->v_least);
    v.batch = c->batch;
    v.kv_heads = c->kv_heads;
    v.max_seq = c->max_seq;
    v.dim = c->dim;
    return ROTOR_B200_OK;
}

static int load_units(Cache4Load& p) {
    const uint32_t quads = (p.begin + p.span + 3) / 4 - p.begin / 4;
    const uint64_t units = (uint64_t)p.c.kv_heads * quads * (p.c.dim / 8);
    if (units > 0x7fffff00u) return ROTOR_B200_ERR_SHAPE;
    p.units = (uint32_t)units;
    p.per_row = FastDiv(p.c.dim / 8);
    p.quads = FastDiv(quads);
    return ROTOR_B200_OK;
}

int launch_cache4_expand(const Cache4Expand& r, cudaStream_t st) {
    Cache4Load p = {};
    p.c = r.c;
    p.dst[0] = r.k;
    p.dst[1] = r.v;
    p.span = r.span;
    p.seq = r.seq;
    p.window = r.window;
    p.negate = r.negate;
    p.past = r.past;
    p.past_out = r.past_out;
    if (const int e = load_units(p)) return e;
    const dim3 grid((p.units + C4_THREADS - 1) / C4_THREADS, p.c.batch, 2);
    return r.half ? launch_chained(cache4_load_kernel<__half, true>, grid, C4_THREADS, 0, st, 1, p)
                  : launch_chained(cache4_load_kernel<__nv_bfloat16, true>, grid, C4_THREADS, 0, st, 1, p);
}

}  // namespace rb

using namespace rb;

extern "C" {

int rotor_b200_cache4_append(const rotor_b200_cache4* cache, const void* k, const void* v, int dtype, const int64_t* k_strides_host,
                             const int64_t* v_strides_host, int seq, int past, const int32_t* past_len, void* stream) {
    Cache4Store p;
    if (const int e = cache4_view(cache, p.c)) return e;
    RB_REQUIRE(k && v && k_strides_host && v_strides_host && dtype >= ROTOR_B200_F32 && dtype <= ROTOR_B200_F16 && seq > 0 && past >= 0);
    RB_REQUIRE(seq <= p.c.max_seq && (past_len || past <= p.c.max_seq - seq));
    const int64_t* strides[2] = {k_strides_host, v_strides_host};
    const int size = dtype == ROTOR_B200_F32 ? 4 : 2;
    p.src[0] = k;
    p.src[1] = v;
    for (int i = 0; i < 2; ++i) {
        const int64_t* s = strides[i];
        RB_REQUIRE(s[0] >= 0 && s[1] >= 0 && s[2] >= 0 && (uintptr_t)p.src[i] % size == 0);
        p.sb[i] = s[0];
        p.ss[i] = s[1];
        p.sh[i] = s[2];
        p.wide[i] = (((uintptr_t)p.src[i] | (uintptr_t)((s[0] | s[1] | s[2]) * size)) & 15) == 0;
    }
    // quads of positions that a sequence's rows can lie in, wherever it starts
    const uint32_t quads = past_len ? (seq + 6) / 4 : (past + seq + 3) / 4 - past / 4;
    const uint64_t units = (uint64_t)quads * p.c.kv_heads * (p.c.dim / 8);
    p.seq = seq;
    if (units > 0x7fffff00u) return ROTOR_B200_ERR_SHAPE;
    p.past = Past{past_len, past, p.c.max_seq};
    p.units = (uint32_t)units;
    p.per_row = FastDiv(p.c.dim / 8);
    p.heads = FastDiv(p.c.kv_heads);
    const dim3 grid((p.units + C4_THREADS - 1) / C4_THREADS, p.c.batch, 2);
    const cudaStream_t st = as_stream(stream);
    switch (dtype) {
        case ROTOR_B200_F32: return launch_chained(cache4_store_kernel<float>, grid, C4_THREADS, 0, st, 1, p);
        case ROTOR_B200_BF16: return launch_chained(cache4_store_kernel<__nv_bfloat16>, grid, C4_THREADS, 0, st, 1, p);
        default: return launch_chained(cache4_store_kernel<__half>, grid, C4_THREADS, 0, st, 1, p);
    }
}

int rotor_b200_cache4_read(const rotor_b200_cache4* cache, int begin, int end, void* k, void* v, int dtype, void* stream) {
    Cache4Load p = {};
    if (const int e = cache4_view(cache, p.c)) return e;
    RB_REQUIRE(k && v && dtype >= ROTOR_B200_F32 && dtype <= ROTOR_B200_F16 && begin >= 0 && end > begin && end <= p.c.max_seq);
    RB_REQUIRE((((uintptr_t)k | (uintptr_t)v) & 15) == 0);
    p.dst[0] = k;
    p.dst[1] = v;
    p.whole = (((uintptr_t)k | (uintptr_t)v) & 31) == 0;
    p.begin = begin;
    p.span = end - begin;
    if (const int e = load_units(p)) return e;
    const dim3 grid((p.units + C4_THREADS - 1) / C4_THREADS, p.c.batch, 2);
    const cudaStream_t st = as_stream(stream);
    switch (dtype) {
        case ROTOR_B200_F32: return launch_chained(cache4_load_kernel<float, false>, grid, C4_THREADS, 0, st, 1, p);
        case ROTOR_B200_BF16: return launch_chained(cache4_load_kernel<__nv_bfloat16, false>, grid, C4_THREADS, 0, st, 1, p);
        default: return launch_chained(cache4_load_kernel<__half, false>, grid, C4_THREADS, 0, st, 1, p);
    }
}

}  // extern "C"
