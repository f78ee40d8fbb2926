// Attention straight over the 4-bit cache (layout: cache4.cuh), for single tokens and portions of a few.
//   score(i, j) = scale q_i . k_j,   j <= pos_i = past + i,   pos_i - j < window if window > 0
//   out_i = sum_j e^(score - top) v_j / (sum_j e^(score - top) + e^(sink - top))
// with k_j = m + s code per group g of 32 columns, so that
//   q . k_j = sum_g s_jg (q_g . code_jg) + sum_g m_jg (sum of q_g)      and      out = sum_g (sum_j (p_j s_jg) code_jg + sum_j p_j m_jg).
//
// Codes are multiplied as they are: a code in the low bits of a float16 is the (subnormal) number code 2^-24, exactly, and one AND makes
// two of them; in the next four bits it is code 2^-20.  No code is converted, and nothing of a cached row is rounded.  The queries of
// 16-bit types are exact in the other operand (a row is scaled by a power of two into float16's range; columns whose codes lie four bits
// higher by another 1/16), float32 queries are split into two terms (2^-22 of the value).  The weights p_j s_jg are rounded to float16
// (2^-12 of the weight; in float32 calls two terms again).  Scores, maxima, sums and outputs are float32.
//
// The shift of the softmax is the running maximum of score + log2(largest s_jg of the row), not of the score: p s is then at most 1 times
// the shift's slack whatever the values' size is, and stays in float16's range.
//
// A warp takes tiles of 16 positions and keeps eight (R = 1) or sixteen (R = 2) query rows of one KV head (row = token x query head of the
// group): scores by m16n8k16 with queries as rows and positions as columns, whose result is the operand that the second product
// (columns of V as rows, queries as columns) takes, without an exchange between lanes.
#include <cmath>

#include "cache4.cuh"

namespace rb {

constexpr int A4_WARPS = 8, A4_THREADS = 32 * A4_WARPS;
constexpr float A4_SLACK = 8.f;   // a new maximum below the old one plus this (in powers of two) leaves the shift where it is
constexpr float A4_LIFT = 7.f;    // weights are at most 2^(A4_SLACK + A4_LIFT), and use float16's range down to 2^-24

struct Attend4 {
    Cache4View c;
    const void* q;
    size_t qb, qs, qh;  // strides of sequence, token and head, in elements
    int dtype, wide;
    void* out;          // [batch][seq][heads][dim]
    float* part;        // [batch][kv_heads][rows][splits][dim + 4]: sums, shift, mass of a split
    const float* sinks;
    Past past;
    int heads, group, seq, rows, window, splits;
    float scale2;       // scale log2(e)
};

__device__ __forceinline__ float a4_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void a4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float2 half2_of(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

// N bytes at an address that is a multiple of the largest power of two that divides N (up to 16), as words.
template <int N>
struct Bytes {
    static constexpr int W = (N + 3) / 4;
    uint32_t w[W];
    __device__ __forceinline__ void load(const void* p) {
        if constexpr (N % 16 == 0) {
#pragma unroll
            for (int i = 0; i < N / 16; ++i) {
                const uint4 v = __ldcg(reinterpret_cast<const uint4*>(p) + i);
                w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
        } else if constexpr (N % 8 == 0) {
#pragma unroll
            for (int i = 0; i < N / 8; ++i) {
                const uint2 v = __ldcg(reinterpret_cast<const uint2*>(p) + i);
                w[2 * i] = v.x, w[2 * i + 1] = v.y;
            }
        } else if constexpr (N % 4 == 0) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) w[i] = __ldcg(reinterpret_cast<const uint32_t*>(p) + i);
        } else {
            static_assert(N % 2 == 0, "16-bit pieces");
#pragma unroll
            for (int i = 0; i < W; ++i) w[i] = 0;
#pragma unroll
            for (int i = 0; i < N / 2; ++i) w[i / 2] |= (uint32_t)__ldcg(reinterpret_cast<const unsigned short*>(p) + i) << (16 * (i & 1));
        }
    }
    // the 16-bit piece i
    __device__ __forceinline__ uint32_t piece(int i) const { return w[i >> 1] >> (16 * (i & 1)) & 0xffffu; }
};

// What a lane (g = lane / 4, t = lane % 4) needs of a tile: column c of the scores' part u is position 4 (c / 2) + 2 u + c % 2, so that a
// lane's four scores of a row are those of positions 4 t .. 4 t + 3, in order.
template <int NG>
struct Tile4 {
    Bytes<4 * NG> k[2];                 // part t of the key rows 4 (g / 2) + 2 u + g % 2
    Bytes<2 * NG> v[4];                 // part g of the value rows 4 t + i
    Bytes<8 * NG> ks, vs, vm;           // rows 4 t .. 4 t + 3
    uint32_t km[2];                     // two groups' m of the key rows of k[]
    __device__ __forceinline__ void load(const Cache4View& c, size_t row0, int g, int t) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const size_t r = row0 + 4 * (g >> 1) + 2 * u + (g & 1);
            k[u].load(c.codes[0] + r * (16 * NG) + t * 4 * NG);
            const __half* m = c.least[0] + r * NG;
            // the matrix instruction that multiplies the m takes a pair of groups per lane (see the queries' sums)
            const int pair = NG > 4 ? 2 * t : 2 * (t & 1);
            const unsigned short* mu = reinterpret_cast<const unsigned short*>(m) + pair;
            if constexpr (NG % 2 == 0)
                km[u] = pair < NG ? __ldcg(reinterpret_cast<const uint32_t*>(mu)) : 0u;
            else
                km[u] = (pair < NG ? __ldcg(mu) : 0u) | (uint32_t)(pair + 1 < NG ? __ldcg(mu + 1) : 0u) << 16;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i].load(c.codes[1] + (row0 + 4 * t + i) * (16 * NG) + g * 2 * NG);
        ks.load(c.step[0] + (row0 + 4 * t) * NG);
        vs.load(c.step[1] + (row0 + 4 * t) * NG);
        vm.load(c.least[1] + (row0 + 4 * t) * NG);
    }
    static __device__ __forceinline__ float half_at(const Bytes<8 * NG>& b, int i) {
        const float2 f = half2_of(b.w[i >> 1]);
        return i & 1 ? f.y : f.x;
    }
};

template <int NG, int R>
struct Attend4Smem {
    static constexpr int D = 32 * NG, Q = 8 * R, OS = D + 4;  // (a row of sums is four floats longer: lanes of a quad on other banks)
    float sums[A4_WARPS][Q][OS];
    float shift[A4_WARPS][Q], mass[A4_WARPS][Q];
};
template <int NG, int R, int TERMS>
struct Attend4Query {
    uint4 frag[NG][TERMS][R][32];  // the queries as operands: per lane a0, a2 (or a1, a3) of a group's two steps of 16 columns
    float top[NG][8 * R], sum[NG][8 * R];
};

template <int NG, int R, int TERMS>
__global__ void __launch_bounds__(A4_THREADS) attend4_kernel(const __grid_constant__ Attend4 p) {
    constexpr int D = 32 * NG, Q = 8 * R;
    using Smem = Attend4Smem<NG, R>;
    using Query = Attend4Query<NG, R, TERMS>;
    extern __shared__ __align__(16) unsigned char a4_raw[];
    Query& sq = *reinterpret_cast<Query*>(a4_raw);
    Smem& sm = *reinterpret_cast<Smem*>(a4_raw);  // (takes the queries' place at the end)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int blocks = (p.rows + Q - 1) / Q;
    const int hk = blockIdx.x / blocks, r0 = (blockIdx.x - hk * blocks) * Q, b = blockIdx.z, split = blockIdx.y;
    pdl_wait();
    pdl_trigger();

    const int past = past_of(p.past, b, p.c.max_seq), last_row = min(r0 + Q, p.rows) - 1;
    const int lo_block = first_visible(past + r0 / p.group, 0, p.window);
    const int hi_block = min(past + last_row / p.group, p.c.max_seq - 1);
    const int tile0 = lo_block / 16, tiles = hi_block / 16 + 1 - tile0;
    const int per = (max(tiles, 0) + p.splits - 1) / p.splits;
    const int first = tile0 + split * per, end = min(first + per, tile0 + tiles);

    // ---- queries: warp j makes the operands of group j
    float qv[R][8], inv_fs[R];
    int lo[R], hi[R];
#pragma unroll
    for (int h = 0; h < R; ++h) {
        const int row = r0 + g + 8 * h, token = min(row, last_row) / p.group, head = hk * p.group + min(row, last_row) - token * p.group;
        lo[h] = first_visible(past + token, 0, p.window);
        hi[h] = row <= last_row ? min(past + token, p.c.max_seq - 1) : -1;
        float top = 0.f;
        if (warp < NG) {
            const size_t at = (size_t)b * p.qb + (size_t)token * p.qs + (size_t)head * p.qh + 32 * warp + 8 * t;
            if (p.dtype == ROTOR_B200_F32)
                load8(static_cast<const float*>(p.q) + at, p.wide, qv[h]);
            else if (p.dtype == ROTOR_B200_BF16)
                load8(static_cast<const __nv_bfloat16*>(p.q) + at, p.wide, qv[h]);
            else
                load8(static_cast<const __half*>(p.q) + at, p.wide, qv[h]);
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                top = fmaxf(top, fabsf(qv[h][n]));
                sum += qv[h][n];
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                sum += __shfl_xor_sync(0xffffffffu, sum, o);
            }
            if (t == 0) {
                sq.top[warp][g + 8 * h] = top;
                sq.sum[warp][g + 8 * h] = sum;
            }
        }
    }
    __syncthreads();
    uint32_t sum_hi[R], sum_lo[R];  // operands: sums of the queries over the groups' columns, as two terms
#pragma unroll
    for (int h = 0; h < R; ++h) {
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < NG; ++j) top = fmaxf(top, sq.top[j][g + 8 * h]);
        // a power of two that takes the row's largest value to 2^14 .. 2^15 (none for rows of zeros, infinities and NaN)
        const int e = (__float_as_int(top) >> 23) - 127;
        const bool scaled = top > 0.f && e < 128;
        const int up = scaled ? min(14 - e, 100) : 0;
        const float fs = __int_as_float((127 + up) << 23);
        inv_fs[h] = __int_as_float((127 - up) << 23);
        if (warp < NG) {
            float x[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) x[n] = qv[h][n] * (n & 1 ? fs * 0.0625f : fs);
#pragma unroll
            for (int term = 0; term < TERMS; ++term) {
                const uint4 f = make_uint4(pack_half(x[0], x[4]), pack_half(x[2], x[6]), pack_half(x[1], x[5]), pack_half(x[3], x[7]));
                sq.frag[warp][term][h][lane] = f;
                if (TERMS > 1) {
                    const float2 a = half2_of(f.x), c = half2_of(f.y), d = half2_of(f.z), w = half2_of(f.w);
                    x[0] -= a.x, x[4] -= a.y, x[2] -= c.x, x[6] -= c.y, x[1] -= d.x, x[5] -= d.y, x[3] -= w.x, x[7] -= w.y;
                }
            }
        }
        const int pair = NG > 4 ? 2 * t : 2 * (t & 1);
        const float f6 = fs * 0.015625f;  // (the sum of 32 columns is up to 2^20 and has to fit as well)
        const float s0 = pair < NG ? sq.sum[pair][g + 8 * h] * f6 : 0.f, s1 = pair + 1 < NG ? sq.sum[pair + 1][g + 8 * h] * f6 : 0.f;
        const uint32_t big = pack_half(s0, s1);
        const float2 bf = half2_of(big);
        const uint32_t rest = pack_half(s0 - bf.x, s1 - bf.y);
        if (NG > 4) {
            sum_hi[h] = big;
            sum_lo[h] = rest;
        } else {  // up to four groups: lanes 0 and 1 of a quad hold the first terms, 2 and 3 the second ones
            sum_hi[h] = t < 2 ? big : rest;
            sum_lo[h] = 0u;
        }
    }
    __syncthreads();

    float shift[R], mass[R], low_sum[R][NG];
    float o[R][2 * NG][4];
#pragma unroll
    for (int h = 0; h < R; ++h) {
        shift[h] = -INFINITY;
        mass[h] = 0.f;
#pragma unroll
        for (int j = 0; j < NG; ++j) low_sum[h][j] = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
            for (int n = 0; n < 4; ++n) o[h][i][n] = 0.f;
    }
    const size_t head_row = ((size_t)b * p.c.kv_heads + hk) * p.c.max_seq;
    for (int tile = first + warp; tile < end; tile += A4_WARPS) {
        Tile4<NG> x;
        x.load(p.c, head_row + (size_t)tile * 16, g, t);

        // ---- scores of 8 R rows x 16 positions: lane's four positions of row g (and g + 8)
        float sc[R][4];
#pragma unroll
        for (int h = 0; h < R; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[h][i] = 0.f;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            float acc[2][4] = {};
            const uint32_t w0 = x.k[0].w[j], w1 = x.k[1].w[j];
#pragma unroll
            for (int term = 0; term < TERMS; ++term) {
                const uint4 fa = sq.frag[j][term][0][lane];
                const uint4 fb = R > 1 ? sq.frag[j][term][R - 1][lane] : make_uint4(0u, 0u, 0u, 0u);
                a4_mma(acc[0], fa.x, fb.x, fa.y, fb.y, w0 & 0x000f000fu, w0 >> 8 & 0x000f000fu);
                a4_mma(acc[1], fa.x, fb.x, fa.y, fb.y, w1 & 0x000f000fu, w1 >> 8 & 0x000f000fu);
                a4_mma(acc[0], fa.z, fb.z, fa.w, fb.w, w0 & 0x00f000f0u, w0 >> 8 & 0x00f000f0u);
                a4_mma(acc[1], fa.z, fb.z, fa.w, fb.w, w1 & 0x00f000f0u, w1 >> 8 & 0x00f000f0u);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float s = Tile4<NG>::half_at(x.ks, i * NG + j);
#pragma unroll
                for (int h = 0; h < R; ++h) sc[h][i] = fmaf(s, acc[i >> 1][2 * h + (i & 1)], sc[h][i]);
            }
        }
        float low[2][4] = {};
#pragma unroll
        for (int u = 0; u < 2; ++u)
            a4_mma(low[u], sum_hi[0], R > 1 ? sum_hi[R - 1] : 0u, NG > 4 ? sum_lo[0] : 0u, NG > 4 && R > 1 ? sum_lo[R - 1] : 0u, x.km[u],
                   NG > 4 ? x.km[u] : 0u);

        // ---- largest step of each position's value row, as a power of two
        float ls[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float m = 5.9604645e-8f;  // the smallest float16 above zero
#pragma unroll
            for (int j = 0; j < NG; ++j) m = fmaxf(m, Tile4<NG>::half_at(x.vs, i * NG + j));
            ls[i] = __log2f(m);
        }
        const int pos = tile * 16 + 4 * t;
        float tmax[R];
        bool higher = false;
#pragma unroll
        for (int h = 0; h < R; ++h) {
            const float f = p.scale2 * inv_fs[h];
            tmax[h] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sc[h][i] = (sc[h][i] * 16777216.f + low[i >> 1][2 * h + (i & 1)] * 64.f) * f;
                if (pos + i < lo[h] || pos + i > hi[h]) sc[h][i] = -INFINITY;
                tmax[h] = fmaxf(tmax[h], sc[h][i] + ls[i]);
            }
            higher |= tmax[h] - A4_LIFT > shift[h] + A4_SLACK;
        }
        if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
            for (int h = 0; h < R; ++h) {
                float m = tmax[h];
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                m = fmaxf(shift[h], m - A4_LIFT);
                const float alpha = m == shift[h] ? 1.f : a4_exp2(shift[h] - m);
                shift[h] = m;
                mass[h] *= alpha;
#pragma unroll
                for (int j = 0; j < NG; ++j) low_sum[h][j] *= alpha;
                // the sums' columns are query rows 2 t and 2 t + 1
                const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * t), a1 = __shfl_sync(0xffffffffu, alpha, 8 * t + 4);
#pragma unroll
                for (int i = 0; i < 2 * NG; ++i) {
                    o[h][i][0] *= a0;
                    o[h][i][1] *= a1;
                    o[h][i][2] *= a0;
                    o[h][i][3] *= a1;
                }
            }
        }
#pragma unroll
        for (int h = 0; h < R; ++h) {
            const float m = shift[h] == -INFINITY ? 0.f : shift[h];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sc[h][i] = a4_exp2(sc[h][i] - m);
                mass[h] += sc[h][i];
            }
        }

        // ---- sums over the positions
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const uint32_t y01 = x.v[0].piece(j) | x.v[1].piece(j) << 16, y23 = x.v[2].piece(j) | x.v[3].piece(j) << 16;
            float s[4], m[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[i] = Tile4<NG>::half_at(x.vs, i * NG + j);
                m[i] = Tile4<NG>::half_at(x.vm, i * NG + j);
            }
#pragma unroll
            for (int h = 0; h < R; ++h) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[i] = sc[h][i] * s[i];
                    low_sum[h][j] = fmaf(sc[h][i], m[i], low_sum[h][j]);
                }
#pragma unroll
                for (int term = 0; term < TERMS; ++term) {
                    const uint32_t b0 = pack_half(w[0], w[1]), b1 = pack_half(w[2], w[3]);
                    a4_mma(o[h][2 * j], y01 & 0x000f000fu, y01 & 0x00f000f0u, y23 & 0x000f000fu, y23 & 0x00f000f0u, b0, b1);
                    a4_mma(o[h][2 * j + 1], y01 >> 8 & 0x000f000fu, y01 >> 8 & 0x00f000f0u, y23 >> 8 & 0x000f000fu, y23 >> 8 & 0x00f000f0u, b0,
                           b1);
                    if (TERMS > 1) {
                        const float2 f0 = half2_of(b0), f1 = half2_of(b1);
                        w[0] -= f0.x, w[1] -= f0.y, w[2] -= f1.x, w[3] -= f1.y;
                    }
                }
            }
        }
    }

    // ---- the warps' sums are joined in shared memory
    __syncthreads();  // (the last query operand has been read)
#pragma unroll
    for (int h = 0; h < R; ++h) {
#pragma unroll
        for (int n = 1; n < 4; n <<= 1) {
            mass[h] += __shfl_xor_sync(0xffffffffu, mass[h], n);
#pragma unroll
            for (int j = 0; j < NG; ++j) low_sum[h][j] += __shfl_xor_sync(0xffffffffu, low_sum[h][j], n);
        }
        if (t == 0) {
            sm.shift[warp][8 * h + g] = shift[h];
            sm.mass[warp][8 * h + g] = mass[h];
        }
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            // columns 32 j + 4 g .. + 3 of query rows 2 t and 2 t + 1; sums of codes four bits higher are 16 times too large
            const float l0 = __shfl_sync(0xffffffffu, low_sum[h][j], 8 * t), l1 = __shfl_sync(0xffffffffu, low_sum[h][j], 8 * t + 4);
            constexpr float c0 = 16777216.f, c1 = 1048576.f;
            const float(&a)[4] = o[h][2 * j], (&c)[4] = o[h][2 * j + 1];
            *reinterpret_cast<float4*>(&sm.sums[warp][8 * h + 2 * t][32 * j + 4 * g]) =
                make_float4(fmaf(a[0], c0, l0), fmaf(a[2], c1, l0), fmaf(c[0], c0, l0), fmaf(c[2], c1, l0));
            *reinterpret_cast<float4*>(&sm.sums[warp][8 * h + 2 * t + 1][32 * j + 4 * g]) =
                make_float4(fmaf(a[1], c0, l1), fmaf(a[3], c1, l1), fmaf(c[1], c0, l1), fmaf(c[3], c1, l1));
        }
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < Q * (D / 4); idx += A4_THREADS) {
        const int r = idx / (D / 4), c4 = idx - r * (D / 4), row = r0 + r;
        if (row >= p.rows) break;
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int w = 0; w < A4_WARPS; ++w) top = fmaxf(top, sm.shift[w][r]);
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        const float ref = top == -INFINITY ? 0.f : top;  // (a warp without a visible position: its zeros times zero; NaN stays)
#pragma unroll
        for (int w = 0; w < A4_WARPS; ++w) {
            const float f = a4_exp2(sm.shift[w][r] - ref);
            const float4 v = *reinterpret_cast<const float4*>(&sm.sums[w][r][4 * c4]);
            total = fmaf(f, sm.mass[w][r], total);
            y.x = fmaf(f, v.x, y.x), y.y = fmaf(f, v.y, y.y), y.z = fmaf(f, v.z, y.z), y.w = fmaf(f, v.w, y.w);
        }
        float* part = p.part + (((size_t)(b * p.c.kv_heads + hk) * p.rows + row) * p.splits + split) * (D + 4);
        *reinterpret_cast<float4*>(part + 4 * c4) = y;
        if (c4 == 0) *reinterpret_cast<float2*>(part + D) = make_float2(top, total);
    }
}

__device__ __forceinline__ void store4(void* out, int dtype, size_t at, float4 y) {
    if (dtype == ROTOR_B200_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = y;
    } else if (dtype == ROTOR_B200_BF16) {
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(out) + at) = float4_to_bf16x4(y);
    } else {
        *reinterpret_cast<uint2*>(static_cast<__half*>(out) + at) = make_uint2(pack_half(y.x, y.y), pack_half(y.z, y.w));
    }
}

// Joins the splits of a query row: a warp per row and 128 columns.
__global__ void __launch_bounds__(32) attend4_join_kernel(const __grid_constant__ Attend4 p) {
    pdl_wait();
    pdl_trigger();
    const int D = p.c.dim, row = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
    const float* part = p.part + ((size_t)(b * p.c.kv_heads + hk) * p.rows + row) * p.splits * (D + 4);
    const int token = row / p.group, head = hk * p.group + row - token * p.group;
    float top = -INFINITY;
    for (int s = 0; s < p.splits; ++s) top = fmaxf(top, __ldcg(part + (size_t)s * (D + 4) + D));
    const float sink = p.sinks ? __ldg(p.sinks + head) * 1.4426950408889634f : -INFINITY;
    const float ref = fmaxf(top, sink) == -INFINITY ? 0.f : fmaxf(top, sink);
    for (int c = 4 * threadIdx.x; c < D; c += 128) {
        float total = a4_exp2(sink - ref);
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s = 0; s < p.splits; ++s) {
            const float* q = part + (size_t)s * (D + 4);
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(q + D));
            const float4 v = __ldcg(reinterpret_cast<const float4*>(q + c));
            const float f = a4_exp2(ml.x - ref);
            total = fmaf(f, ml.y, total);
            y.x = fmaf(f, v.x, y.x), y.y = fmaf(f, v.y, y.y), y.z = fmaf(f, v.z, y.z), y.w = fmaf(f, v.w, y.w);
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;  // (a row that sees no position: zeros)
        store4(p.out, p.dtype, (((size_t)b * p.seq + token) * p.heads + head) * D + c, make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
    }
}

struct Attend4Plan {
    int splits, per_block;  // query rows of a block
    size_t part_bytes;
};

static Attend4Plan attend4_plan(const Cache4View& c, int rows, int reach) {
    Attend4Plan a;
    const int ng = c.dim / C4_GROUP;
    a.per_block = rows > 8 && ng <= 4 ? 16 : 8;
    const long long blocks = (long long)c.batch * c.kv_heads * ((rows + a.per_block - 1) / a.per_block);
    const long long tiles = (reach + 15) / 16 + 1;
    long long splits = (2LL * fused_sm_count() + blocks - 1) / blocks;
    const long long most = (tiles + A4_WARPS - 1) / A4_WARPS;  // a tile per warp
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    a.splits = (int)splits;
    a.part_bytes = (size_t)c.batch * c.kv_heads * rows * splits * (c.dim + 4) * sizeof(float);
    return a;
}

template <int NG, int R, int TERMS>
static int attend4_go(const Attend4& a, const Attend4Plan& plan, cudaStream_t st) {
    constexpr size_t s1 = sizeof(Attend4Smem<NG, R>), s2 = sizeof(Attend4Query<NG, R, TERMS>), smem = s1 > s2 ? s1 : s2;
    static PerDevice<bool> once;
    if (!once.here()) {
        RB_CUDA(cudaFuncSetAttribute(attend4_kernel<NG, R, TERMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        once.here() = true;
    }
    const dim3 grid(a.c.kv_heads * ((a.rows + plan.per_block - 1) / plan.per_block), a.splits, a.c.batch);
    if (const int e = launch_chained(attend4_kernel<NG, R, TERMS>, grid, A4_THREADS, smem, st, 1, a)) return e;
    return launch_chained(attend4_join_kernel, dim3(a.rows, a.c.kv_heads, a.c.batch), 32, 0, st, 1, a);
}

template <int NG>
static int attend4_pick(const Attend4& a, const Attend4Plan& plan, cudaStream_t st) {
    const bool f32 = a.dtype == ROTOR_B200_F32;
    if constexpr (NG <= 4)
        if (plan.per_block == 16) return f32 ? attend4_go<NG, 2, 2>(a, plan, st) : attend4_go<NG, 2, 1>(a, plan, st);
    return f32 ? attend4_go<NG, 1, 2>(a, plan, st) : attend4_go<NG, 1, 1>(a, plan, st);
}

static int attend4_check(const rotor_b200_cache4* cache, Cache4View& c, int heads, int seq, int longest) {
    if (const int e = cache4_view(cache, c)) return e;
    RB_REQUIRE(heads > 0 && heads % c.kv_heads == 0 && seq > 0 && longest >= 0);
    if ((long long)seq * (heads / c.kv_heads) > (1 << 24) || heads > 65535) return ROTOR_B200_ERR_SHAPE;
    return ROTOR_B200_OK;
}

// The most positions that the queries of a call see between them.
static int attend4_reach(const Cache4View& c, int seq, int longest, int window) {
    long long reach = (long long)longest + seq;
    if (window > 0 && reach > (long long)window + seq) reach = (long long)window + seq;
    return (int)(reach < c.max_seq ? reach : c.max_seq);
}

}  // namespace rb

using namespace rb;

extern "C" {

size_t rotor_b200_cache4_attend_workspace_bytes(const rotor_b200_cache4* cache, int heads, int seq, int longest, int window) {
    Cache4View c;
    if (attend4_check(cache, c, heads, seq, longest)) return 0;
    return attend4_plan(c, seq * (heads / c.kv_heads), attend4_reach(c, seq, longest, window)).part_bytes;
}

int rotor_b200_cache4_attend(const rotor_b200_cache4* cache, const void* q, int dtype, const int64_t* q_strides_host, int heads, int seq,
                             int past, const int32_t* past_len, int longest, float scale, int window, const float* sinks, void* out,
                             void* workspace, size_t workspace_bytes, void* stream) {
    Attend4 a;
    if (const int e = attend4_check(cache, a.c, heads, seq, longest)) return e;
    RB_REQUIRE(q && q_strides_host && out && workspace && dtype >= ROTOR_B200_F32 && dtype <= ROTOR_B200_F16 && past >= 0 && window >= 0);
    RB_REQUIRE(seq <= a.c.max_seq && (past_len || past <= a.c.max_seq - seq));
    const int64_t* s = q_strides_host;
    const int size = dtype == ROTOR_B200_F32 ? 4 : 2;
    RB_REQUIRE(s[0] >= 0 && s[1] >= 0 && s[2] >= 0 && (uintptr_t)q % size == 0 && (((uintptr_t)out | (uintptr_t)workspace) & 15) == 0);
    a.q = q;
    a.qb = s[0];
    a.qs = s[1];
    a.qh = s[2];
    a.dtype = dtype;
    a.wide = (((uintptr_t)q | (uintptr_t)((s[0] | s[1] | s[2]) * size)) & 15) == 0;
    a.out = out;
    a.part = static_cast<float*>(workspace);
    a.sinks = sinks;
    a.past = Past{past_len, past};
    a.heads = heads;
    a.group = heads / a.c.kv_heads;
    a.seq = seq;
    a.rows = seq * a.group;
    a.window = window;
    a.scale2 = scale * 1.4426950408889634f;
    const Attend4Plan plan = attend4_plan(a.c, a.rows, attend4_reach(a.c, seq, past_len ? longest : past, window));
    if (plan.part_bytes > workspace_bytes) return ROTOR_B200_ERR_WORKSPACE;
    a.splits = plan.splits;
    const cudaStream_t st = as_stream(stream);
    switch (a.c.dim / C4_GROUP) {
        case 1: return attend4_pick<1>(a, plan, st);
        case 2: return attend4_pick<2>(a, plan, st);
        case 3: return attend4_pick<3>(a, plan, st);
        case 4: return attend4_pick<4>(a, plan, st);
        case 6: return attend4_pick<6>(a, plan, st);
        default: return attend4_pick<8>(a, plan, st);
    }
}

}  // extern "C"
