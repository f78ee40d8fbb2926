// Keys and values of one layer in 4 bits.
//
// A row (one position of one KV head) is cut into groups of 32 columns.  Of a group are held m, its smallest value, and
// s = (largest - smallest) / 15, both float16, and per column the code of 0 .. 15 nearest to (x - m) / s (the even one of two as
// near); a code stands for m + s code.  128 columns take 80 bytes: 3.2 times less than bf16, 6.4 times less than float32.
//
// Everything lies in the order in which the attention's matrix instructions take it (m16n8k16, lane = 4 g + t), so that a lane loads its
// part in whole pieces and nothing is moved between lanes.  NG = dim / 32 groups, j a group; inside a KV head's positions:
//   key codes    [position][t][j] words: columns 32 j + 8 t .. + 7, column 8 t + n in bits 4 n .. 4 n + 3
//   key s, m     [position][j]
//   value codes  tiles of 16 positions; [j][lane][position % 4] 16-bit words, t = position % 16 / 4: columns 32 j + 4 g .. + 3, column
//                4 g + n in bits 4 n .. 4 n + 3; two groups' words of a lane are neighbours (value_at)
//   value s, m   [position / 4][j][position % 4]
#pragma once
#include <cuda_fp16.h>

#include "decoder.cuh"

namespace rb {

constexpr int C4_GROUP = 32;
constexpr int C4_POSITIONS = 16;    // max_seq is a multiple of this: a tile of the attention ends inside the cache
constexpr float C4_MOST = 65504.f;  // magnitudes above the largest float16 are stored as that

// Place of group j's word of position % 16 = r, part g, in a tile of value codes, in 16-bit words.
__host__ __device__ __forceinline__ int value_at(int NG, int j, int g, int r) {
    const int lane = 4 * g + (r >> 2);
    return (j < NG / 2 * 2 ? j / 2 * 256 + lane * 8 + j % 2 * 4 : NG / 2 * 256 + lane * 4) + (r & 3);
}

struct Cache4View {
    uint8_t* codes[2];              // keys, values: [batch][kv_heads][max_seq][dim / 2]
    __half *step[2], *least[2];     // s and m: [batch][kv_heads][max_seq][dim / 32]
    int batch, kv_heads, max_seq, dim;
};

// x / d for x below 2^31, by a multiplication (a division by a number known at launch costs about twenty instructions).
struct FastDiv {
    uint32_t d, mul, shift;
    __host__ explicit FastDiv(uint32_t n = 1) : d(n), shift(0) {
        while ((1ull << shift) < n) ++shift;
        mul = (uint32_t)((((1ull << shift) - n) << 32) / n + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t x) const { return (__umulhi(x, mul) + x) >> shift; }
};

// Where sequence b of a call starts: a number for all, or one per sequence in device memory, taken as at most `most`.
struct Past {
    const int* each;
    int all, most;
};
__device__ __forceinline__ int past_of(const Past& p, int b) { return p.each ? min(max(__ldcg(p.each + b), 0), p.most) : p.all; }

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The cluster's barrier, and loads from the shared memory of its CTA `rank`.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_at(const float* local, unsigned rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    return a;
}
__device__ __forceinline__ float2 cluster_load2(const float* local, unsigned rank) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(cluster_at(local, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float4 cluster_load4(const float* local, unsigned rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(cluster_at(local, rank))
                 : "memory");
    return v;
}

__device__ __forceinline__ float type_load(const float* p) { return *p; }
__device__ __forceinline__ float type_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float type_load(const __half* p) { return __half2float(*p); }

// Eight neighbours as float32; `wide`: the address is a multiple of 16 bytes.
__device__ __forceinline__ void load8(const float* p, bool wide, float (&x)[8]) {
    if (wide) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
}
template <typename T2, typename T>
__device__ __forceinline__ void load8_half(const T* p, bool wide, float (&x)[8]) {
    if (wide) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const T2 h = *reinterpret_cast<const T2*>(&w[i]);
            x[2 * i] = type_load(&h.x);
            x[2 * i + 1] = type_load(&h.y);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = type_load(p + i);
    }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, bool wide, float (&x)[8]) { load8_half<__nv_bfloat162>(p, wide, x); }
__device__ __forceinline__ void load8(const __half* p, bool wide, float (&x)[8]) { load8_half<__half2>(p, wide, x); }

__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
    const uint2 a = float4_to_bf16x4(make_float4(x[0], x[1], x[2], x[3])), b = float4_to_bf16x4(make_float4(x[4], x[5], x[6], x[7]));
    *reinterpret_cast<uint4*>(p) = make_uint4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// The same for outputs of finite rows: what rounding takes above 65504 is that (NaN stays).
__device__ __forceinline__ uint32_t pack_half_finite(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void store8(__half* p, const float (&x)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_half(x[0], x[1]), pack_half(x[2], x[3]), pack_half(x[4], x[5]), pack_half(x[6], x[7]));
}

int cache4_view(const rotor_b200_cache4* c, Cache4View& v);  // checks the description


// The first `span` positions of every sequence and head as dense rows [batch][kv_heads][span][dim], bf16 or float16, as the prompt attention
// of `seq` tokens reads them: zeros behind a sequence's last position, nothing where no query looks, keys times -1 with `negate`.  past goes to past_out too.
struct Cache4Expand {
    Cache4View c;
    void *k, *v;
    int half, span, seq, window, negate;
    Past past;
    int* past_out;
};
int launch_cache4_expand(const Cache4Expand& r, cudaStream_t st);

// Attention of prompts over those rows.  Sequence b holds past_len[b] positions (at most max_seq) before its tokens; positions from max_seq
// on do not exist.  Rows up to 127 behind a sequence's last one are read and multiplied by zero: they have to hold numbers.  The keys hold
// the scale's sign.  No stride of an extent above one is zero.
struct PromptAttn {
    const void *q, *k, *v;
    size_t q_seq, q_row, q_head;  // strides in elements; rows begin at multiples of 16 bytes
    const int* past_len;
    const float* sinks;           // [heads], or null
    void* out;                    // [batch][seq][heads][dim]
    int half, batch, seq, heads, kv_heads, dim, span, max_seq, window;
    float scale;
};
bool prompt_attn_supported(int batch, int heads, int kv_heads, int dim, int span);
int launch_prompt_attn(const PromptAttn& p, cudaStream_t st);

}  // namespace rb
