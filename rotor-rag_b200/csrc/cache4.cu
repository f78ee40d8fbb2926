// The 4-bit cache is written and read back (layout: cache4.cuh).  Both directions move bytes: of a bf16 row of 128 columns 256 bytes
// on the dense side and 80 in the cache.  A thread takes eight neighbouring columns, which are one word of a key row or two 16-bit words
// of a value tile, and four threads a group; threads run along rows.
#include "cache4.cuh"

namespace rb {

constexpr int C4_THREADS = 256;

// Where eight columns (c8 of a row) of a position lie: their word of the keys, or two 16-bit words of the values, `next` apart (parts g and
// g + 1 of a tile), and their group's s and m.
struct Place {
    uint16_t* codes;
    size_t group;
    int next;
    __device__ __forceinline__ Place(const Cache4View& c, int part, int b, uint32_t h, int pos, uint32_t c8) {
        const int NG = c.dim / C4_GROUP, j = c8 >> 2, t = c8 & 3;
        const size_t head = ((size_t)b * c.kv_heads + h) * c.max_seq;
        if (part == 0) {
            codes = reinterpret_cast<uint16_t*>(c.codes[0]) + (head + pos) * (NG * 8) + (t * NG + j) * 2;
            group = (head + pos) * NG + j;
            next = 1;
        } else {
            codes = reinterpret_cast<uint16_t*>(c.codes[1]) + (head + (pos & ~15)) * (NG * 8) + value_at(NG, j, 2 * t, pos & 15);
            group = (head + (pos & ~3)) * NG + j * 4 + (pos & 3);
            next = value_at(NG, j, 1, 0) - value_at(NG, j, 0, 0);
        }
    }
};

struct Cache4Store {
    Cache4View c;
    const void* src[2];
    size_t sb[2], ss[2], sh[2];  // strides of sequence, position and head, in elements
    bool wide[2];                // rows begin at multiples of 16 bytes
    Past past;
    uint32_t units;              // seq * kv_heads * dim / 8
    FastDiv per_row, heads;
};

// s of a group.  The definition rounds the quotient in 64 bits to float32 and then to float16.  float32 arithmetic gives the same
// float16 unless its result is within a few of its own steps of a border between two float16 numbers.
__device__ __forceinline__ __half group_step(float low, float high) {
    const float q = __fdiv_rn(high - low, 15.f);
    const int low_bits = __float_as_int(q) & 0x1fff;  // of a normal float16 these are cut off, and 0x1000 is the border
    if (high > low && (q < 6.2e-5f || (low_bits >= 0x1000 - 4 && low_bits <= 0x1000 + 4)))
        return __float2half_rn((float)(((double)high - (double)low) / 15.0));
    return __float2half_rn(q);
}

template <typename T>
__global__ void __launch_bounds__(C4_THREADS) cache4_store_kernel(const __grid_constant__ Cache4Store p) {
    pdl_wait();
    pdl_trigger();
    const uint32_t u = blockIdx.x * C4_THREADS + threadIdx.x;
    const int b = blockIdx.y, part = blockIdx.z;
    const bool on = u < p.units;
    const uint32_t row = p.per_row.div(on ? u : 0), c8 = (on ? u : 0) - row * p.per_row.d;
    const uint32_t i = p.heads.div(row), h = row - i * p.heads.d;
    float x[8];
    load8(static_cast<const T*>(p.src[part]) + (size_t)b * p.sb[part] + (size_t)i * p.ss[part] + (size_t)h * p.sh[part] + c8 * 8, p.wide[part], x);
    // (minimum and maximum pass over NaN; a group of nothing else holds zeros)
    float low = INFINITY, high = -INFINITY;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
        if (x[n] == x[n]) x[n] = fminf(fmaxf(x[n], -C4_MOST), C4_MOST);
        low = fminf(low, x[n]);
        high = fmaxf(high, x[n]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    if (low > high) low = high = 0.f;
    const __half sh = group_step(low, high), mh = __float2half_rn(low);
    const float s = __half2float(sh), m = __half2float(mh);
    const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
    uint32_t word = 0;
    bool close = false;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
        const float q = fminf(fmaxf((x[n] - m) * inv, 0.f), 15.f), code = rintf(q);  // (NaN: 0)
        close |= fabsf(fabsf(q - code) - 0.5f) < 2e-5f;
        word |= (uint32_t)(int)code << (4 * n);
    }
    // The quotient in float32 is off by less than 1e-5: next to a border between two codes it is taken in 64 bits.
    if (close) {
        word = 0;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const double q = ((double)x[n] - (double)m) / (double)s;
            word |= (uint32_t)(int)fmin(fmax(rint(q), 0.0), 15.0) << (4 * n);
        }
    }
    const int pos = past_of(p.past, b) + (int)i;
    if (!on || pos >= p.c.max_seq) return;
    const Place w(p.c, part, b, h, pos, c8);
    if (part == 0) {
        *reinterpret_cast<uint32_t*>(w.codes) = word;
    } else {
        w.codes[0] = (uint16_t)word;
        w.codes[w.next] = (uint16_t)(word >> 16);
    }
    if ((c8 & 3) == 0) {
        p.c.step[part][w.group] = sh;
        p.c.least[part][w.group] = mh;
    }
}

struct Cache4Load {
    Cache4View c;
    void* dst[2];
    int begin, span;
    uint32_t units;  // kv_heads * span * dim / 8
    FastDiv per_row, positions;
    // rows for a prompt
    int seq, window;
    Past past;
    int* past_out;
};

template <typename T, bool PROMPT>
__global__ void __launch_bounds__(C4_THREADS) cache4_load_kernel(const __grid_constant__ Cache4Load p) {
    pdl_wait();
    pdl_trigger();
    const uint32_t u = blockIdx.x * C4_THREADS + threadIdx.x;
    const int b = blockIdx.y, part = blockIdx.z;
    if (u >= p.units) return;
    const uint32_t row = p.per_row.div(u), c8 = u - row * p.per_row.d;
    const uint32_t h = p.positions.div(row), pos = p.begin + row - h * p.positions.d;
    bool there = true;
    if constexpr (PROMPT) {
        // the attention reads tiles of 128 positions from the first one its first query sees: a head's rows end in zeros, and so begin
        // the rows that a tile at the end of the head before reaches into
        const int past = past_of(p.past, b), limit = min(past + p.seq, p.c.max_seq);
        if (p.past_out && u == 0 && part == 0) p.past_out[b] = past;
        if ((int)pos >= limit + 128 || ((int)pos < first_visible(past, 0, p.window) && pos >= 128)) return;
        there = (int)pos < limit;
    }
    float x[8];
    uint32_t word = 0;
    float s = 0.f, m = 0.f;
    if (there) {
        const Place w(p.c, part, b, h, pos, c8);
        word = part == 0 ? *reinterpret_cast<const uint32_t*>(w.codes) : w.codes[0] | (uint32_t)w.codes[w.next] << 16;
        s = __half2float(p.c.step[part][w.group]);
        m = __half2float(p.c.least[part][w.group]);
    }
#pragma unroll
    for (int n = 0; n < 8; ++n) x[n] = fmaf((float)(word >> (4 * n) & 15u), s, m);
    if constexpr (PROMPT) {
#pragma unroll
        for (int n = 0; n < 8; ++n) x[n] = fminf(x[n], C4_MOST);  // (m + 15 s may lie a rounding above the largest float16)
    }
    store8(static_cast<T*>(p.dst[part]) + (((size_t)b * p.c.kv_heads + h) * p.span + (pos - p.begin)) * p.c.dim + c8 * 8, x);
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
    const uint64_t units = (uint64_t)p.c.kv_heads * p.span * (p.c.dim / 8);
    if (units > 0x7fffff00u) return ROTOR_B200_ERR_SHAPE;
    p.units = (uint32_t)units;
    p.per_row = FastDiv(p.c.dim / 8);
    p.positions = FastDiv(p.span);
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
    const uint64_t units = (uint64_t)seq * p.c.kv_heads * (p.c.dim / 8);
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
