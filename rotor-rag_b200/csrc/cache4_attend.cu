// Attention straight over the 4-bit cache (layout: cache4.cuh), for single tokens and portions of a few.
//   score(i, j) = scale q_i . k_j,   j <= pos_i = past + i,   pos_i - j < window if window > 0
//   out_i = sum_j e^(score - top) v_j / (sum_j e^(score - top) + e^(sink - top))
// with k_j = m + s code per group g of 32 columns, so that
//   q . k_j = sum_g s_jg (q_g . code_jg) + sum_g m_jg (sum of q_g)      and      out = sum_g (sum_j (p_j s_jg) code_jg + sum_j p_j m_jg).
//
// Codes are multiplied as they are: a code in the low bits of a float16 is the (subnormal) number code 2^-24, exactly, and one AND makes
// two of them; in the next four bits it is code 2^-20.  No code is converted, and nothing of a cached row is rounded.  The queries of
// 16-bit types are exact in the other operand (a row is scaled by a power of two into float16's range; columns whose codes lie four bits
// higher by another 1/16), float32 queries are split into two terms (2^-22 of the value).  The weights p_j are rounded to float16 and so
// are their products with s_jg (2^-11 each, or 2^-25 where that is more, the largest weight of a row being 2^7 or more; the sum of weights
// takes them as rounded).  In float32 calls both are two terms, the second held 2^10 times as large and with sums of its own, so that it keeps
// its bits where the first is near float16's smallest numbers: 2^-22 of a weight, and 2^-35 of the largest.  There a warp multiplies s by a
// power of two that takes the largest it has seen to between 2^-4 and 2, so that products keep these bits at values of any size.  (One sum for
// both terms was off by 2e-5 of the weighted sums for values of 1e-5 and nearly equal scores, where this is within 2^-17, and took 58.5 us where
// this takes 64.5: 64 sequences behind 1024 .. 4095 positions, 64/8 heads of 128.)
// Scores, maxima, sums and outputs are float32.  Matrix instructions cut their sums off instead of rounding them, which shows after many
// of them in a row, and align their products as if a subnormal number had the smallest normal exponent: with codes in the lowest four bits
// a sum is off by 1.7e-7 of its terms' size, four bits higher by 3e-9 (as with the codes as normal numbers).  float32 calls begin every
// tile's sums at zero and add them up outside, and shift all codes to the higher place.
//
// A warp takes tiles of 16 positions and keeps eight (R = 1) or sixteen (R = 2) query rows of one KV head (row = token x query head of the
// group).  Both products have the codes as their 16-row operand: S = K Q^T (positions x queries) and O^T = V^T P (columns x queries);
// two 8 x 8 transposes (movmatrix) turn the weights from the one's result into the other's operand.  One more instruction per tile sums
// p m over the groups and, in a row of ones, p itself.
//
// Tiles travel by cp.async into a ring of the warp's own (no barrier, and the loads in flight do not depend on what the registers hold):
// a tile of 128 columns is 2560 bytes, five copies a lane.
#include <cmath>

#include "cache4.cuh"

namespace rb {

constexpr float A4_LOW = -3.4028235e38f;  // the shift of rows that have seen nothing: no finite score is below
constexpr float A4_SECOND = 1024.f;  // second terms of weights are held this many times as large
constexpr int A4_MOST_UP = 14;       // with two terms s is multiplied by up to 2^14
constexpr int A4_NEAR_ONE = 4;       // ... and by none where the largest is between 2^-4 and 2, as it is for values around 1
constexpr int A4_JOIN = 256;      // threads of the join
constexpr int A4_SORTED = 128;    // most sequences that are taken by their length
constexpr int A4_CLUSTER = 8;     // most splits that are joined inside a cluster
// Dense keys (and values) of a prompt at a time, unless one sequence has more: the rows take 3.2 times the cache's memory, and sequences after
// one another keep the workspace at 1 GiB.  (That much is 0.4 ms of writing alone: a launch more does not show.)
constexpr size_t A4_DENSE = (size_t)1 << 29;

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
    int by_length;      // CTAs take the sequences from the longest to the shortest
    float scale2;       // scale log2(e)
};

__device__ __forceinline__ void a4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float2 half2_of(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

// N bytes of shared memory at an address that is a multiple of the largest power of two that divides N (up to 16), as words.
template <int N>
struct Bytes {
    static constexpr int W = (N + 3) / 4;
    uint32_t w[W];
    __device__ __forceinline__ void load(const unsigned char* p) {
        if constexpr (N % 16 == 0) {
#pragma unroll
            for (int i = 0; i < N / 16; ++i) {
                const uint4 v = reinterpret_cast<const uint4*>(p)[i];
                w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
        } else if constexpr (N % 8 == 0) {
#pragma unroll
            for (int i = 0; i < N / 8; ++i) {
                const uint2 v = reinterpret_cast<const uint2*>(p)[i];
                w[2 * i] = v.x, w[2 * i + 1] = v.y;
            }
        } else if constexpr (N % 4 == 0) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
        } else {
            static_assert(N % 2 == 0, "16-bit pieces");
#pragma unroll
            for (int i = 0; i < W; ++i) w[i] = 0;
#pragma unroll
            for (int i = 0; i < N / 2; ++i) w[i / 2] |= (uint32_t)reinterpret_cast<const unsigned short*>(p)[i] << (16 * (i & 1));
        }
    }
    __device__ __forceinline__ float half_at(int i) const {
        const float2 f = half2_of(w[i >> 1]);
        return i & 1 ? f.y : f.x;
    }
};

__device__ __forceinline__ uint32_t turned(uint32_t v) {  // the 8 x 8 matrix of 16-bit numbers, transposed
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float two_to(int e) { return __int_as_float((127 + e) << 23); }
__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ uint32_t as_word(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A tile in shared memory: key codes, value codes, then s and m of the keys and of the values.
template <int NG>
struct Tile4 {
    static constexpr int V = 256 * NG, KS = 512 * NG, KM = 544 * NG, VS = 576 * NG, VM = 608 * NG, BYTES = 640 * NG;
    // 16-byte pieces: 16 NG of each kind of codes, 8 NG of s and m; pieces lane + 32 r of a lane's rounds
    static constexpr int CODE_ROUNDS = (NG + 1) / 2, REST_ROUNDS = (NG + 3) / 4;
    const unsigned char *k, *v, *rest[REST_ROUNDS];  // where this lane's pieces of tile 0 of the head are
    __device__ __forceinline__ Tile4(const Cache4View& c, size_t head_row, int lane) {
        k = c.codes[0] + head_row * (16 * NG) + lane * 16;
        v = c.codes[1] + head_row * (16 * NG) + lane * 16;
        const __half* kinds[4] = {c.step[0], c.least[0], c.step[1], c.least[1]};
#pragma unroll
        for (int r = 0; r < REST_ROUNDS; ++r) {
            const int piece = lane + 32 * r, kind = min(piece / (2 * NG), 3);
            const __half* base = kind == 0 ? kinds[0] : kind == 1 ? kinds[1] : kind == 2 ? kinds[2] : kinds[3];
            rest[r] = reinterpret_cast<const unsigned char*>(base + head_row * NG) + (piece - kind * 2 * NG) * 16;
        }
    }
    __device__ __forceinline__ void fetch(int tile, uint32_t dst, int lane) const {
#pragma unroll
        for (int r = 0; r < CODE_ROUNDS; ++r) {
            if (NG % 2 == 0 || lane + 32 * r < 16 * NG) {
                copy16(dst + (lane + 32 * r) * 16, k + (size_t)tile * V + 512 * r);
                copy16(dst + V + (lane + 32 * r) * 16, v + (size_t)tile * V + 512 * r);
            }
        }
#pragma unroll
        for (int r = 0; r < REST_ROUNDS; ++r)
            if (NG % 4 == 0 || lane + 32 * r < 8 * NG) copy16(dst + KS + (lane + 32 * r) * 16, rest[r] + (size_t)tile * (32 * NG));
    }
};

// Every fourth code of a word (of a pair of 16-bit words), as two float16 numbers: 2^-24 (codes 0 and 2) or 2^-20 (1 and 3) times the code;
// EXACT: 2^-20 for all.
template <bool EXACT, int I>
__device__ __forceinline__ uint32_t codes_of(uint32_t w) {
    if constexpr (EXACT) return (I == 0 ? w << 4 : I == 1 ? w : I == 2 ? w >> 4 : w >> 8) & 0x00f000f0u;
    return (I < 2 ? w : w >> 8) & (I % 2 ? 0x00f000f0u : 0x000f000fu);
}
constexpr float A4_LOW_CODE = 16777216.f, A4_HIGH_CODE = 1048576.f;  // 2^24, 2^20

template <int NG, int R, int TERMS, int W>
struct A4Cfg {
    static constexpr int D = 32 * NG, Q = 8 * R;
    static constexpr int STAGES = NG >= 6 ? 2 : 3;
    static constexpr int OS = D + 4;             // floats between a row's sums and the next: lanes of a quad on other banks
    static constexpr bool KEEP = NG * R * TERMS <= 4;  // the queries' operands stay in registers
    // queries as operands: per lane two pairs of a group's two steps of 16 columns; largest values and sums of the groups
    static constexpr int FRAG = 0, TOPS = FRAG + NG * TERMS * R * 512, SUMS = TOPS + NG * Q * 4, RING = SUMS + NG * Q * 4;
    static constexpr int RING_BYTES = W * STAGES * Tile4<NG>::BYTES;
    // at the end, over the ring: sums of the warps' rows, shifts, masses; then the CTA's rows for the cluster
    static constexpr int O = RING, SHIFT = O + W * Q * OS * 4, MASS = SHIFT + W * Q * 4, ROWS = MASS + W * Q * 4;
    static constexpr int END = ROWS + Q * OS * 4, SMEM = END > RING + RING_BYTES ? END : RING + RING_BYTES;
};

__device__ __forceinline__ void store4(void* out, int dtype, size_t at, float4 y) {
    if (dtype == ROTOR_B200_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = y;
    } else if (dtype == ROTOR_B200_BF16) {
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(out) + at) = float4_to_bf16x4(y);
    } else {
        *reinterpret_cast<uint2*>(static_cast<__half*>(out) + at) = make_uint2(pack_half_finite(y.x, y.y), pack_half_finite(y.z, y.w));
    }
}

// Four columns of a query row from the sums y, their mass and shift.  A row that sees no position gives zeros.
__device__ __forceinline__ void finish4(const Attend4& p, int b, int hk, int row, int col, float4 y, float mass, float shift) {
    const int token = row / p.group, head = hk * p.group + row - token * p.group;
    if (p.sinks) {
        const float sink = __ldg(p.sinks + head) * 1.4426950408889634f, top = fmaxf(shift, sink), mine = fast_exp2(shift - top);
        mass = fmaf(mass, mine, fast_exp2(sink - top));
        y.x *= mine, y.y *= mine, y.z *= mine, y.w *= mine;
    }
    const float inv = mass == 0.f ? 0.f : 1.f / mass;
    store4(p.out, p.dtype, (((size_t)b * p.seq + token) * p.heads + head) * p.c.dim + col, make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
}

template <int NG, int R, int TERMS, int W>
__global__ void __launch_bounds__(32 * W, (NG * R <= 4 ? 16 : 8) / W) attend4_kernel(const __grid_constant__ Attend4 p) {
    using C = A4Cfg<NG, R, TERMS, W>;
    constexpr bool EXACT = TERMS > 1;
    // A new maximum below the old one plus SLACK (powers of two) leaves the shift where it is, and weights are at most 2^(lift + SLACK).  p s is
    // below 2^15 for s below 2, and for larger s the lift is smaller; with two terms p s is below 2^5, so that 2^10 times that is a float16 too.
    constexpr float SLACK = EXACT ? 4.f : 7.f, LIFT = EXACT ? 0.f : 7.f;
    constexpr int THREADS = 32 * W, OWN = (NG + W - 1) / W;  // groups whose query operands a warp makes
    using T = Tile4<NG>;
    constexpr int D = C::D, Q = C::Q, S = C::STAGES;
    extern __shared__ __align__(128) unsigned char a4_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int blocks = (p.rows + Q - 1) / Q, block = blockIdx.x / p.splits, split = blockIdx.x - block * p.splits;
    const int hk = block / blocks, r0 = (block - hk * blocks) * Q, last_row = min(r0 + Q, p.rows) - 1;
    pdl_wait();
    pdl_trigger();
    int b = blockIdx.y;
    if (p.by_length) {  // the longest sequences first: this CTA's is the one with blockIdx.y longer ones
        int* lengths = reinterpret_cast<int*>(a4_raw + C::RING);
        int& chosen = lengths[A4_SORTED];
        int own = 0;
        if (threadIdx.x < p.c.batch) lengths[threadIdx.x] = own = past_of(p.past, threadIdx.x);
        __syncthreads();
        if (threadIdx.x < p.c.batch) {
            int longer = 0;
            for (int i = 0; i < p.c.batch; ++i) longer += lengths[i] > own || (lengths[i] == own && i < (int)threadIdx.x);
            if (longer == b) chosen = threadIdx.x;
        }
        __syncthreads();
        b = chosen;
        __syncthreads();  // (tiles are copied here next)
    }

    // ---- queries: warp j loads group j (and j + W), which does not wait for the sequence's length
    float qv[R][OWN][8];
#pragma unroll
    for (int h = 0; h < R; ++h) {
        const int row = min(r0 + g + 8 * h, last_row), token = row / p.group, head = hk * p.group + row - token * p.group;
        const size_t at = (size_t)b * p.qb + (size_t)token * p.qs + (size_t)head * p.qh + 8 * t;
#pragma unroll
        for (int k = 0; k < OWN; ++k) {
            const int j = warp + k * W;
            if (j < NG) {
                if (p.dtype == ROTOR_B200_F32)
                    load8(static_cast<const float*>(p.q) + at + 32 * j, p.wide, qv[h][k]);
                else if (p.dtype == ROTOR_B200_BF16)
                    load8(static_cast<const __nv_bfloat16*>(p.q) + at + 32 * j, p.wide, qv[h][k]);
                else
                    load8(static_cast<const __half*>(p.q) + at + 32 * j, p.wide, qv[h][k]);
            }
        }
    }

    // ---- the first tiles
    const int past = past_of(p.past, b);
    const int pos0 = past + r0 / p.group, pos1 = past + last_row / p.group;  // positions of the block's first and last row
    const int seen0 = first_visible(pos0, 0, p.window), seen1 = min(pos1, p.c.max_seq - 1);  // what some row sees
    const int tile0 = seen0 / 16, tiles = max(seen1 / 16 + 1 - tile0, 0);
    const int per = (tiles + p.splits - 1) / p.splits;
    const int first = tile0 + split * per + warp, end = min(tile0 + (split + 1) * per, tile0 + tiles);
    const T source(p.c, ((size_t)b * p.c.kv_heads + hk) * p.c.max_seq, lane);
    unsigned char* ring = a4_raw + C::RING + warp * S * T::BYTES;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
        if (first + s * W < end) source.fetch(first + s * W, ring_at + s * T::BYTES, lane);
        copy_commit();
    }

    // ---- the queries' operands
    uint4* frags = reinterpret_cast<uint4*>(a4_raw + C::FRAG);  // [j][term][h][lane]
    float(*tops)[Q] = reinterpret_cast<float(*)[Q]>(a4_raw + C::TOPS);
    float(*sums)[Q] = reinterpret_cast<float(*)[Q]>(a4_raw + C::SUMS);
    float fa[R][2];
    int lo[R][2], hi[R][2];  // visible positions of query rows 2 t and 2 t + 1 (+ 8 h)
#pragma unroll
    for (int h = 0; h < R; ++h) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = r0 + 8 * h + 2 * t + e, pos = past + min(row, last_row) / p.group;
            lo[h][e] = first_visible(pos, 0, p.window);
            hi[h][e] = min(pos, p.c.max_seq - 1);  // (rows past the last one repeat it, and are not kept)
        }
#pragma unroll
        for (int k = 0; k < OWN; ++k) {
            const int j = warp + k * W;
            if (j < NG) {
                float top = 0.f, sum = 0.f;
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    top = fmaxf(top, fabsf(qv[h][k][n]));
                    sum += qv[h][k][n];
                }
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) {
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    sum += __shfl_xor_sync(0xffffffffu, sum, o);
                }
                if (t == 0) {
                    tops[j][g + 8 * h] = top;
                    sums[j][g + 8 * h] = sum;
                }
            }
        }
    }
    __syncthreads();
    uint32_t sum_hi[R], sum_lo[R];  // operands: sums of the queries over the groups' columns, as two terms
#pragma unroll
    for (int h = 0; h < R; ++h) {
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < NG; ++j) top = fmaxf(top, tops[j][g + 8 * h]);
        // a power of two that takes the row's largest value to 2^14 .. 2^15 (none for rows of zeros, infinities and NaN)
        const int e = (__float_as_int(top) >> 23) - 127;
        const int up = top > 0.f && e < 128 ? min(14 - e, 100) : 0;
        const float fs = __int_as_float((127 + up) << 23), back = p.scale2 * __int_as_float((127 - up) << 23);
        fa[h][0] = __shfl_sync(0xffffffffu, back, 8 * t);
        fa[h][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
#pragma unroll
        for (int k = 0; k < OWN; ++k) {
            const int j = warp + k * W;
            if (j < NG) {
                float x[8];
#pragma unroll
                for (int n = 0; n < 8; ++n) x[n] = qv[h][k][n] * (n & 1 && !EXACT ? fs * 0.0625f : fs);
#pragma unroll
                for (int term = 0; term < TERMS; ++term) {
                    const uint4 f = make_uint4(pack_half(x[0], x[4]), pack_half(x[2], x[6]), pack_half(x[1], x[5]), pack_half(x[3], x[7]));
                    frags[((j * TERMS + term) * R + h) * 32 + lane] = f;
                    if (TERMS > 1) {
                        const float2 a = half2_of(f.x), c = half2_of(f.y), d = half2_of(f.z), w = half2_of(f.w);
                        x[0] -= a.x, x[4] -= a.y, x[2] -= c.x, x[6] -= c.y, x[1] -= d.x, x[5] -= d.y, x[3] -= w.x, x[7] -= w.y;
                    }
                }
            }
        }
        // up to four groups: lanes 0 and 1 of a quad hold the first terms of two groups, 2 and 3 the second ones
        const int pair = NG > 4 ? 2 * t : 2 * (t & 1);
        const float f6 = fs * 0.015625f;  // (the sum of 32 columns is up to 2^20 and has to fit as well)
        const float s0 = pair < NG ? sums[pair][g + 8 * h] * f6 : 0.f, s1 = pair + 1 < NG ? sums[pair + 1][g + 8 * h] * f6 : 0.f;
        const uint32_t big = pack_half(s0, s1);
        const float2 bf = half2_of(big);
        const uint32_t rest = pack_half(s0 - bf.x, s1 - bf.y);
        sum_hi[h] = NG > 4 || t < 2 ? big : rest;
        sum_lo[h] = NG > 4 ? rest : 0u;
    }
    __syncthreads();
    uint4 kept[C::KEEP ? NG * TERMS * R : 1];
    if constexpr (C::KEEP) {
#pragma unroll
        for (int i = 0; i < NG * TERMS * R; ++i) kept[i] = frags[i * 32 + lane];
    }
    auto frag = [&](int j, int term, int h) {
        const int i = (j * TERMS + term) * R + h;
        return C::KEEP ? kept[C::KEEP ? i : 0] : frags[i * 32 + lane];
    };

    float shift[R][2], o[R][2 * NG][4], rest[R][4];  // rest: row g: sum of p m of group g; row 8 (lanes 0 .. 3): sum of p
    float lift = LIFT;
    float up = (float)(1 << A4_MOST_UP);  // EXACT: what s is multiplied by, a power of two; the sums o are that many times as large
#pragma unroll
    for (int h = 0; h < R; ++h) {
        shift[h][0] = shift[h][1] = A4_LOW;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            rest[h][n] = 0.f;
#pragma unroll
            for (int i = 0; i < 2 * NG; ++i) o[h][i][n] = 0.f;
        }
    }
    auto rescale = [&](int h, float a0, float a1, float f) {
        const float f0 = EXACT ? a0 * f : a0, f1 = EXACT ? a1 * f : a1;
#pragma unroll
        for (int i = 0; i < 2 * NG; ++i) o[h][i][0] *= f0, o[h][i][1] *= f1, o[h][i][2] *= f0, o[h][i][3] *= f1;
        rest[h][0] *= a0, rest[h][1] *= a1, rest[h][2] *= a0, rest[h][3] *= a1;
    };
    const int key_row = 4 * (g >> 1) + (g & 1);  // rows g and g + 8 of the key operand: this position of the tile, and two more
    // tiles that every row sees whole
    const int inner0 = (first_visible(pos1, 0, p.window) + 15) / 16, inner1 = (min(pos0, p.c.max_seq - 1) + 1) / 16;
    int stage = 0;
    for (int tile = first; tile < end; tile += W) {
        copy_wait<S - 2>();
        __syncwarp();
        {
            const int ahead = tile + (S - 1) * W;
            const int into = stage == 0 ? S - 1 : stage - 1;
            if (ahead < end) source.fetch(ahead, ring_at + into * T::BYTES, lane);
            copy_commit();
        }
        const unsigned char* x = ring + stage * T::BYTES;
        stage = stage == S - 1 ? 0 : stage + 1;

        // ---- scores of 16 positions x 8 R rows: lane's positions key_row and key_row + 2, rows 2 t and 2 t + 1 (+ 8 h)
        float sc[R][4];
        {
            Bytes<4 * NG> k0, k1;
            Bytes<2 * NG> s0, s1;
            k0.load(x + key_row * (16 * NG) + t * (4 * NG));
            k1.load(x + (key_row + 2) * (16 * NG) + t * (4 * NG));
            s0.load(x + T::KS + key_row * (2 * NG));
            s1.load(x + T::KS + (key_row + 2) * (2 * NG));
            uint32_t km[2];
            const int pair = NG > 4 ? 2 * t : 2 * (t & 1);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const unsigned short* m = reinterpret_cast<const unsigned short*>(x + T::KM + (key_row + 2 * u) * (2 * NG)) + pair;
                if constexpr (NG % 2 == 0)
                    km[u] = pair < NG ? *reinterpret_cast<const uint32_t*>(m) : 0u;
                else
                    km[u] = (pair < NG ? m[0] : 0u) | (uint32_t)(pair + 1 < NG ? m[1] : 0u) << 16;
            }
#pragma unroll
            for (int h = 0; h < R; ++h) {
                float low[4] = {0.f, 0.f, 0.f, 0.f};
                a4_mma(low, km[0], km[1], NG > 4 ? km[0] : 0u, NG > 4 ? km[1] : 0u, sum_hi[h], sum_lo[h]);
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[h][i] = low[i] * 64.f;
            }
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                const uint32_t w0 = k0.w[j], w1 = k1.w[j];
                constexpr float unit = EXACT ? A4_HIGH_CODE : A4_LOW_CODE;
                const float f0 = s0.half_at(j) * unit, f1 = s1.half_at(j) * unit;
#pragma unroll
                for (int h = 0; h < R; ++h) {
                    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int term = TERMS - 1; term >= 0; --term) {
                        const uint4 f = frag(j, term, h);
                        a4_mma(acc, codes_of<EXACT, 0>(w0), codes_of<EXACT, 0>(w1), codes_of<EXACT, 2>(w0), codes_of<EXACT, 2>(w1), f.x, f.y);
                        a4_mma(acc, codes_of<EXACT, 1>(w0), codes_of<EXACT, 1>(w1), codes_of<EXACT, 3>(w0), codes_of<EXACT, 3>(w1), f.z, f.w);
                    }
                    sc[h][0] = fmaf(f0, acc[0], sc[h][0]);
                    sc[h][1] = fmaf(f0, acc[1], sc[h][1]);
                    sc[h][2] = fmaf(f1, acc[2], sc[h][2]);
                    sc[h][3] = fmaf(f1, acc[3], sc[h][3]);
                }
            }
        }
#pragma unroll
        for (int h = 0; h < R; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[h][i] *= fa[h][i & 1];

        // ---- the values' s; where one is 2 or more (bit 14 of a float16) weights, or with two terms s, have to be smaller
        Bytes<8 * NG> vs;
        vs.load(x + T::VS + t * (8 * NG));
        if (tile < inner0 || tile >= inner1) {
#pragma unroll
            for (int h = 0; h < R; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int pos = tile * 16 + key_row + (i & 2);
                    if (pos < lo[h][i & 1] || pos > hi[h][i & 1]) sc[h][i] = -INFINITY;
                }
            // (what lies in places that no row sees does not count)
            const int at = tile * 16 + 4 * t;
            auto seen = [&](int pos) { return pos >= seen0 && pos <= seen1 ? 0xffffu : 0u; };
            const uint32_t m01 = seen(at) | seen(at + 1) << 16, m23 = seen(at + 2) | seen(at + 3) << 16;
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                vs.w[2 * j] &= m01;
                vs.w[2 * j + 1] &= m23;
            }
        }
        uint32_t any = 0;
        if constexpr (EXACT) {
            // the largest, in both halves of the word (s is no negative number: floats in the order of their bits)
            uint32_t most = 0u;
#pragma unroll
            for (int i = 0; i < 2 * NG; ++i) most = __vmaxu2(most, vs.w[i]);
            any = as_word(__hmul2(as_half2(most), __float2half2_rn(up)));
        } else {
#pragma unroll
            for (int i = 0; i < 2 * NG; ++i) any |= vs.w[i];
        }
        bool higher = false;
#pragma unroll
        for (int h = 0; h < R; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) higher |= fmaxf(sc[h][e], sc[h][e + 2]) > shift[h][e] + (SLACK + lift);
        if (__any_sync(0xffffffffu, higher || (any & 0x40004000u))) {
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < 4 * NG; ++i) most = fmaxf(most, vs.half_at(i));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const int exponent = (__float_as_int(most) >> 23) - 127;  // (of zero: -127)
            const float now = EXACT ? lift : fminf(lift, LIFT - (float)max(exponent, 0));
            float f = 1.f;
            if constexpr (EXACT) {
                const float best = two_to(exponent >= -A4_NEAR_ONE && exponent <= 0 ? 0 : min(-exponent, A4_MOST_UP));
                if (best < up) {
                    f = best * two_to(127 - (__float_as_int(up) >> 23));
                    up = best;
                }
            }
#pragma unroll
            for (int h = 0; h < R; ++h) {
                float alpha[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float m = fmaxf(sc[h][e], sc[h][e + 2]);
#pragma unroll
                    for (int n = 4; n < 32; n <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, n));
                    m = fmaxf(shift[h][e] + (lift - now), m - now);
                    alpha[e] = fast_exp2(shift[h][e] - m);
                    shift[h][e] = m;
                }
                rescale(h, alpha[0], alpha[1], f);
            }
            lift = now;
        }
        if constexpr (EXACT) {
            if (up != 1.f) {
                const __half2 f = __float2half2_rn(up);
#pragma unroll
                for (int i = 0; i < 2 * NG; ++i) vs.w[i] = as_word(__hmul2(as_half2(vs.w[i]), f));
            }
        }

        // ---- weights, turned into the operand of the second product: row g of the queries, positions 4 t .. 4 t + 3
        uint32_t pw[R][TERMS][2];
#pragma unroll
        for (int h = 0; h < R; ++h) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float e0 = fast_exp2(sc[h][2 * u] - shift[h][0]), e1 = fast_exp2(sc[h][2 * u + 1] - shift[h][1]);
                const uint32_t w = pack_half(e0, e1);
                pw[h][0][u] = turned(w);
                if (TERMS > 1) {
                    const float2 f = half2_of(w);
                    pw[h][TERMS - 1][u] = turned(pack_half((e0 - f.x) * A4_SECOND, (e1 - f.y) * A4_SECOND));
                }
            }
        }

        // ---- sums over the positions
        {
            Bytes<8> vm;
            vm.w[0] = vm.w[1] = 0u;
            if (g < NG) vm.load(x + T::VM + t * (8 * NG) + g * 8);
            const uint32_t ones = g == 0 ? 0x3c003c00u : 0u;
#pragma unroll
            for (int h = 0; h < R; ++h) {
                if constexpr (TERMS > 1) {
                    float d[4] = {0.f, 0.f, 0.f, 0.f}, l[4] = {0.f, 0.f, 0.f, 0.f};
                    a4_mma(l, vm.w[0], ones, vm.w[1], ones, pw[h][1][0], pw[h][1][1]);
                    a4_mma(d, vm.w[0], ones, vm.w[1], ones, pw[h][0][0], pw[h][0][1]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) rest[h][i] += fmaf(l[i], 1.f / A4_SECOND, d[i]);
                } else {
                    a4_mma(rest[h], vm.w[0], ones, vm.w[1], ones, pw[h][0][0], pw[h][0][1]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            Bytes<8> y;  // words of positions 4 t, 4 t + 1 and 4 t + 2, 4 t + 3
            y.load(x + T::V + 2 * value_at(NG, j, 0, 0) + lane * (j < NG / 2 * 2 ? 16 : 8));
            const uint32_t a = y.w[0], c = y.w[1];
#pragma unroll
            for (int h = 0; h < R; ++h) {
                const __half2 s0 = as_half2(vs.w[2 * j]), s1 = as_half2(vs.w[2 * j + 1]);
                const __half2 w0 = __hmul2(as_half2(pw[h][0][0]), s0), w1 = __hmul2(as_half2(pw[h][0][1]), s1);
                if constexpr (TERMS > 1) {
                    // the second term holds what the rounding of p s left out, and the second term of p
                    const __half2 many = __float2half2_rn(A4_SECOND), t0 = __hmul2(s0, many), t1 = __hmul2(s1, many);
                    const __half2 l0 = __hfma2(as_half2(pw[h][1][0]), s0, __hfma2(as_half2(pw[h][0][0]), t0, __hneg2(__hmul2(w0, many))));
                    const __half2 l1 = __hfma2(as_half2(pw[h][1][1]), s1, __hfma2(as_half2(pw[h][0][1]), t1, __hneg2(__hmul2(w1, many))));
                    float d[4] = {0.f, 0.f, 0.f, 0.f}, d2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int term = 1; term >= 0; --term) {
                        const uint32_t b0 = as_word(term ? l0 : w0), b1 = as_word(term ? l1 : w1);
                        a4_mma(d, codes_of<EXACT, 0>(a), codes_of<EXACT, 1>(a), codes_of<EXACT, 0>(c), codes_of<EXACT, 1>(c), b0, b1);
                        a4_mma(d2, codes_of<EXACT, 2>(a), codes_of<EXACT, 3>(a), codes_of<EXACT, 2>(c), codes_of<EXACT, 3>(c), b0, b1);
                        if (term) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                d[i] *= 1.f / A4_SECOND;
                                d2[i] *= 1.f / A4_SECOND;
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o[h][2 * j][i] += d[i];
                        o[h][2 * j + 1][i] += d2[i];
                    }
                } else {
                    a4_mma(o[h][2 * j], codes_of<EXACT, 0>(a), codes_of<EXACT, 1>(a), codes_of<EXACT, 0>(c), codes_of<EXACT, 1>(c), as_word(w0), as_word(w1));
                    a4_mma(o[h][2 * j + 1], codes_of<EXACT, 2>(a), codes_of<EXACT, 3>(a), codes_of<EXACT, 2>(c), codes_of<EXACT, 3>(c), as_word(w0),
                           as_word(w1));
                }
            }
        }
    }

    // ---- the warps' sums are joined in shared memory
    copy_wait<0>();
    __syncthreads();  // (every warp has read its last tile: the sums lie over the rings)
    float* all = reinterpret_cast<float*>(a4_raw + C::O);  // [warp][row][OS]
    float(*shifts)[Q] = reinterpret_cast<float(*)[Q]>(a4_raw + C::SHIFT);
    float(*masses)[Q] = reinterpret_cast<float(*)[Q]>(a4_raw + C::MASS);
    const float down = two_to(127 - (__float_as_int(up) >> 23));
#pragma unroll
    for (int h = 0; h < R; ++h) {
        const int r = 8 * h + 2 * t;
        if (g == 0) {
            shifts[warp][r] = shift[h][0];
            shifts[warp][r + 1] = shift[h][1];
            masses[warp][r] = rest[h][2];
            masses[warp][r + 1] = rest[h][3];
        }
        float* to = all + (warp * Q + r) * C::OS + 4 * g;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            // columns 32 j + 4 g .. + 3
            const float l0 = __shfl_sync(0xffffffffu, rest[h][0], 4 * j + t), l1 = __shfl_sync(0xffffffffu, rest[h][1], 4 * j + t);
            const float c0 = EXACT ? A4_HIGH_CODE * down : A4_LOW_CODE, c1 = EXACT ? A4_HIGH_CODE * down : A4_HIGH_CODE;
            const float(&a)[4] = o[h][2 * j], (&c)[4] = o[h][2 * j + 1];
            *reinterpret_cast<float4*>(to + 32 * j) = make_float4(fmaf(a[0], c0, l0), fmaf(a[2], c1, l0), fmaf(c[0], c0, l0), fmaf(c[2], c1, l0));
            *reinterpret_cast<float4*>(to + C::OS + 32 * j) =
                make_float4(fmaf(a[1], c0, l1), fmaf(a[3], c1, l1), fmaf(c[1], c0, l1), fmaf(c[3], c1, l1));
        }
    }
    __syncthreads();
    float* mine = reinterpret_cast<float*>(a4_raw + C::ROWS);  // [row][OS]: sums, shift, mass
    for (int idx = threadIdx.x; idx < Q * (D / 4); idx += THREADS) {
        const int r = idx / (D / 4), c4 = idx - r * (D / 4), row = r0 + r;
        if (row >= p.rows) break;
        float top = A4_LOW, total = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, shifts[w][r]);
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = fast_exp2(shifts[w][r] - top);
            const float4 v = *reinterpret_cast<const float4*>(all + (w * Q + r) * C::OS + 4 * c4);
            total = fmaf(f, masses[w][r], total);
            y.x = fmaf(f, v.x, y.x), y.y = fmaf(f, v.y, y.y), y.z = fmaf(f, v.z, y.z), y.w = fmaf(f, v.w, y.w);
        }
        if (p.splits == 1) {
            finish4(p, b, hk, row, 4 * c4, y, total, top);
            continue;
        }
        if (p.splits <= A4_CLUSTER) {
            *reinterpret_cast<float4*>(mine + r * C::OS + 4 * c4) = y;
            if (c4 == 0) *reinterpret_cast<float2*>(mine + r * C::OS + D) = make_float2(top, total);
            continue;
        }
        float* part = p.part + (((size_t)(b * p.c.kv_heads + hk) * p.rows + row) * p.splits + split) * (D + 4);
        *reinterpret_cast<float4*>(part + 4 * c4) = y;
        if (c4 == 0) *reinterpret_cast<float2*>(part + D) = make_float2(top, total);
    }
    if (p.splits == 1 || p.splits > A4_CLUSTER) return;
    // the CTAs of a cluster are the splits of its rows: each finishes a share of them
    cluster_sync();
    for (int idx = threadIdx.x * p.splits + split; idx < Q * (D / 4); idx += THREADS * p.splits) {
        const int r = idx / (D / 4), c4 = idx - r * (D / 4), row = r0 + r;
        if (row >= p.rows) break;
        float2 sm[A4_CLUSTER];
        float4 v[A4_CLUSTER];
#pragma unroll
        for (int k = 0; k < A4_CLUSTER; ++k)
            if (k < p.splits) {
                sm[k] = cluster_load2(mine + r * C::OS + D, k);
                v[k] = cluster_load4(mine + r * C::OS + 4 * c4, k);
            }
        float top = A4_LOW, total = 0.f;
#pragma unroll
        for (int k = 0; k < A4_CLUSTER; ++k)
            if (k < p.splits) top = fmaxf(top, sm[k].x);
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < A4_CLUSTER; ++k)
            if (k < p.splits) {
                const float f = fast_exp2(sm[k].x - top);
                total = fmaf(f, sm[k].y, total);
                y.x = fmaf(f, v[k].x, y.x), y.y = fmaf(f, v[k].y, y.y), y.z = fmaf(f, v[k].z, y.z), y.w = fmaf(f, v[k].w, y.w);
            }
        finish4(p, b, hk, row, 4 * c4, y, total, top);
    }
    cluster_sync();  // (nobody leaves while its rows are being read)
}

// Joins the splits of a query row where they are more than a cluster: a CTA per row, its threads columns x shares of the splits.
__global__ void __launch_bounds__(A4_JOIN) attend4_join_kernel(const __grid_constant__ Attend4 p) {
    __shared__ float4 s_y[A4_JOIN];
    __shared__ float s_mass[A4_JOIN];
    pdl_wait();
    pdl_trigger();
    const int D = p.c.dim, hk = blockIdx.x / p.rows, row = blockIdx.x - hk * p.rows, b = blockIdx.y;
    const int shares = A4_JOIN / (D / 4), share = threadIdx.x / (D / 4), c = threadIdx.x - share * (D / 4);
    const float* part = p.part + ((size_t)(b * p.c.kv_heads + hk) * p.rows + row) * p.splits * (D + 4);
    float top = A4_LOW;
    for (int s = threadIdx.x & 31; s < p.splits; s += 32) top = fmaxf(top, __ldcg(part + (size_t)s * (D + 4) + D));
    top = warp_max(top);
    float total = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float f, float mass, const float4& v) {
        total = fmaf(f, mass, total);
        y.x = fmaf(f, v.x, y.x), y.y = fmaf(f, v.y, y.y), y.z = fmaf(f, v.z, y.z), y.w = fmaf(f, v.w, y.w);
    };
    if (share < shares) {
#pragma unroll 8
        for (int s = share; s < p.splits; s += shares) {
            const float* q = part + (size_t)s * (D + 4);
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(q + D));
            add(fast_exp2(ml.x - top), ml.y, __ldcg(reinterpret_cast<const float4*>(q + 4 * c)));
        }
    }
    s_y[threadIdx.x] = y;
    s_mass[threadIdx.x] = total;
    __syncthreads();
    if (share > 0) return;
    for (int k = 1; k < shares; ++k) add(1.f, s_mass[k * (D / 4) + c], s_y[k * (D / 4) + c]);
    finish4(p, b, hk, row, 4 * c, y, total, top);
}

struct Attend4Plan {
    bool prompt;             // the cache's rows are made dense (bf16 or float16) in the workspace, for the prompt kernel
    int span, chunk;         // prompt: dense rows of a head, sequences at a time
    size_t dense_bytes;      // of the keys, and of the values
    int splits, per_block, by_length;  // else: CTAs that share a row's positions, query rows of a block, longest sequences first
    size_t bytes;            // of workspace
};

// For sequences that hold up to `longest` positions (each its own number of them: `ragged`).  What is fastest goes by estimates in us:
//   here      two CTAs (R NG > 4: one) are on an SM; a CTA takes about 4 us beside its tiles (lengths and queries arrive, the warps' sums are
//             joined), 0.7 more for a join inside a cluster and 3.5 for the join kernel; a tile of 128 columns of every warp 0.9 us
//             (the rate of the memory), of sixteen query rows 1.5, with a CTA on an SM 0.75
//   prompts   dense rows at about 5 TB/s and 3 us, then a CTA per SM, 9 us and for every 128 keys of its items (two blocks of 128 query rows)
//             1.8, with many items on every SM 2.2 and 1 for an item
// Measured here / as prompts, bf16, heads of 128: 16 tokens of 4 sequences behind 2000 positions, 20/5 heads, 17.5 / 43.1 us, 64 tokens
// 49.1 / 48.2, 256 tokens 148 / 51.7; 16 tokens behind 16000 positions, 64/8 heads, 53 / 246, 64 tokens 232 / 246, 128 tokens 356 / 247;
// 32 sequences, 32/8 heads, behind 500 positions: 16 tokens 52 / 56, 32 tokens 104 / 60, 256 tokens 942 / 155.  Heads of 64, 8 sequences, 16/4
// heads, behind 2000 positions: 64 tokens 37 / 43, 128 tokens 64 / 44.
static Attend4Plan attend4_plan(const Cache4View& c, int dtype, int heads, int seq, int longest, int window, bool boxes, bool ragged) {
    Attend4Plan a = {};
    const int group = heads / c.kv_heads, rows = seq * group, ng = c.dim / C4_GROUP, sms = fused_sm_count();
    const int held = (int)((long long)longest + seq < c.max_seq ? longest + seq : c.max_seq);
    const int reach = window > 0 && held > (long long)window + seq ? window + seq : held;  // what the queries see between them
    a.per_block = rows > 8 ? 16 : 8;
    const long long blocks = (long long)c.batch * c.kv_heads * ((rows + a.per_block - 1) / a.per_block), tiles = (reach + 15) / 16 + 1;
    const bool pair = ng * a.per_block <= 32;
    const long long slots = sms * (pair ? 2 : 1);
    const double tile_us = (!pair ? 0.75 : a.per_block == 16 ? 1.5 : 0.9) * ng / 4;
    double best = 1e30;
    auto consider = [&](long long splits) {
        if (splits < 1 || (splits - 1) * 8 >= tiles) return;
        const double rounds = (double)((blocks * splits + slots - 1) / slots), each = (double)((tiles + splits * 8 - 1) / (splits * 8));
        const double us = rounds * (4.0 + each * tile_us) + (splits == 1 ? 0.0 : splits <= A4_CLUSTER ? 0.7 : 3.5);
        if (us < best) {
            best = us;
            a.splits = (int)splits;
        }
    };
    for (int splits = 1; splits <= A4_CLUSTER; ++splits) consider(splits);
    for (int round = 1; round <= 2; ++round) consider(slots * round / blocks > A4_CLUSTER ? slots * round / blocks : 0);
    consider(slots / blocks > A4_CLUSTER ? (tiles + 7) / 8 : 0);

    a.span = held;
    const size_t each = (size_t)c.kv_heads * a.span * c.dim * 2;
    a.chunk = (int)(each * c.batch <= A4_DENSE ? c.batch : each < A4_DENSE ? A4_DENSE / each : 1);
    a.dense_bytes = round_up(each * a.chunk, 256);
    if (boxes && dtype != ROTOR_B200_F32 && rows > 16 && prompt_attn_supported(a.chunk, heads, c.kv_heads, c.dim, a.span) &&
        (uint64_t)c.kv_heads * a.span * (c.dim / 8) <= 0x7fffff00u) {
        const double most = (reach + 127) / 128, mean = most - 0.5 * (seq < reach ? seq : reach) / 128;  // tiles of keys
        const double dense = 3.0 + (double)c.batch * c.kv_heads * reach * c.dim * 5.25 * 1e-6 / 5.0;
        const int tokens = 2 * (128 / group);
        const long long items = (long long)c.batch * c.kv_heads * ((seq + tokens - 1) / tokens);
        const double one = 1.8 * most, all = (double)((items + sms - 1) / sms) * (1.0 + 2.2 * mean);
        a.prompt = dense + 9.0 + (one > all ? one : all) < best;
    }
    if (a.prompt) {
        a.bytes = 2 * a.dense_bytes + (size_t)a.chunk * sizeof(int);
        return a;
    }
    a.by_length = ragged && c.batch <= A4_SORTED && blocks * a.splits > slots;
    a.bytes = a.splits <= A4_CLUSTER ? 0 : (size_t)c.batch * c.kv_heads * rows * a.splits * (c.dim + 4) * sizeof(float);
    return a;
}

template <int NG, int R, int TERMS, int W>
static int attend4_go(const Attend4& a, cudaStream_t st) {
    constexpr int smem = A4Cfg<NG, R, TERMS, W>::SMEM;
    static PerDevice<bool> once;
    if (!once.here()) {
        RB_CUDA(cudaFuncSetAttribute(attend4_kernel<NG, R, TERMS, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        once.here() = true;
    }
    const bool cluster = a.splits > 1 && a.splits <= A4_CLUSTER;
    const dim3 grid(a.c.kv_heads * ((a.rows + 8 * R - 1) / (8 * R)) * a.splits, a.c.batch);
    const int e = launch_chained(attend4_kernel<NG, R, TERMS, W>, grid, 32 * W, smem, st, cluster ? a.splits : 1, a);
    return e || a.splits <= A4_CLUSTER ? e : launch_chained(attend4_join_kernel, dim3(a.rows * a.c.kv_heads, a.c.batch), A4_JOIN, 0, st, 1, a);
}

template <int NG>
static int attend4_pick(const Attend4& a, const Attend4Plan& plan, cudaStream_t st) {
    const bool f32 = a.dtype == ROTOR_B200_F32;
    if (plan.per_block == 16) return f32 ? attend4_go<NG, 2, 2, 8>(a, st) : attend4_go<NG, 2, 1, 8>(a, st);
    return f32 ? attend4_go<NG, 1, 2, 8>(a, st) : attend4_go<NG, 1, 1, 8>(a, st);
}

// Sequences b .. b + n - 1, or as many as there are.
static Cache4View cache4_part(Cache4View c, int b, int n) {
    const size_t rows = (size_t)b * c.kv_heads * c.max_seq;
    for (int i = 0; i < 2; ++i) {
        c.codes[i] += rows * (c.dim / 2);
        c.step[i] += rows * (c.dim / C4_GROUP);
        c.least[i] += rows * (c.dim / C4_GROUP);
    }
    c.batch = n < c.batch - b ? n : c.batch - b;
    return c;
}

static int attend4_check(const rotor_b200_cache4* cache, Cache4View& c, int dtype, int heads, int seq, int longest, int window) {
    if (const int e = cache4_view(cache, c)) return e;
    RB_REQUIRE(dtype >= ROTOR_B200_F32 && dtype <= ROTOR_B200_F16 && heads > 0 && heads % c.kv_heads == 0);
    RB_REQUIRE(seq > 0 && seq <= c.max_seq && longest >= 0 && window >= 0);
    if ((long long)seq * (heads / c.kv_heads) > (1 << 24) || heads > 65535) return ROTOR_B200_ERR_SHAPE;
    return ROTOR_B200_OK;
}

}  // namespace rb

using namespace rb;

extern "C" {

size_t rotor_b200_cache4_attend_workspace_bytes(const rotor_b200_cache4* cache, int dtype, int heads, int seq, int longest, int window) {
    Cache4View c;
    if (attend4_check(cache, c, dtype, heads, seq, longest, window)) return 0;
    const size_t a = attend4_plan(c, dtype, heads, seq, longest, window, true, true).bytes;
    const size_t b = attend4_plan(c, dtype, heads, seq, longest, window, false, true).bytes;
    return a > b ? a : b > 16 ? b : 16;
}

int rotor_b200_cache4_attend(const rotor_b200_cache4* cache, const void* q, int dtype, const int64_t* q_strides_host, int heads, int seq,
                             int past, const int32_t* past_len, int longest, float scale, int window, const float* sinks, void* out,
                             void* workspace, size_t workspace_bytes, void* stream) {
    Attend4 a;
    if (const int e = attend4_check(cache, a.c, dtype, heads, seq, longest, window)) return e;
    RB_REQUIRE(q && q_strides_host && out && past >= 0 && (past_len || past <= a.c.max_seq - seq));
    const int64_t* s = q_strides_host;
    const int size = dtype == ROTOR_B200_F32 ? 4 : 2;
    RB_REQUIRE(s[0] >= 0 && s[1] >= 0 && s[2] >= 0 && (uintptr_t)q % size == 0 && (((uintptr_t)out | (uintptr_t)workspace) & 15) == 0);
    a.wide = (((uintptr_t)q | (uintptr_t)((s[0] | s[1] | s[2]) * size)) & 15) == 0;
    a.past = Past{past_len, past, longest < a.c.max_seq ? longest : a.c.max_seq};
    // (the prompt kernel copies whole boxes of queries: rows that lie apart)
    const bool boxes = a.wide && (s[0] > 0 || a.c.batch == 1) && (s[1] > 0 || seq == 1) && (s[2] > 0 || heads == 1);
    const Attend4Plan plan = attend4_plan(a.c, dtype, heads, seq, past_len ? longest : past, window, boxes, past_len != nullptr);
    if (plan.bytes > workspace_bytes || (plan.bytes && !workspace)) return ROTOR_B200_ERR_WORKSPACE;
    const cudaStream_t st = as_stream(stream);
    if (plan.prompt) {
        Cache4Expand x;
        x.k = workspace;
        x.v = static_cast<char*>(workspace) + plan.dense_bytes;
        x.half = dtype == ROTOR_B200_F16;
        x.span = plan.span;
        x.seq = seq;
        x.window = window;
        x.negate = scale < 0.f;
        x.past_out = reinterpret_cast<int*>(static_cast<char*>(workspace) + 2 * plan.dense_bytes);
        PromptAttn p;
        p.k = x.k;
        p.v = x.v;
        p.q_seq = s[0];
        p.q_row = s[1];
        p.q_head = s[2];
        p.past_len = x.past_out;
        p.sinks = sinks;
        p.half = x.half;
        p.seq = seq;
        p.heads = heads;
        p.kv_heads = a.c.kv_heads;
        p.dim = a.c.dim;
        p.span = plan.span;
        p.max_seq = a.c.max_seq;
        p.window = window;
        p.scale = scale;
        for (int b = 0; b < a.c.batch; b += plan.chunk) {
            x.c = cache4_part(a.c, b, plan.chunk);
            x.past = Past{past_len ? past_len + b : nullptr, a.past.all, a.past.most};
            p.batch = x.c.batch;
            p.q = static_cast<const uint16_t*>(q) + (size_t)b * s[0];
            p.out = static_cast<uint16_t*>(out) + (size_t)b * seq * heads * a.c.dim;
            if (const int e = launch_cache4_expand(x, st)) return e;
            if (const int e = launch_prompt_attn(p, st)) return e;
        }
        return ROTOR_B200_OK;
    }
    a.q = q;
    a.qb = s[0];
    a.qs = s[1];
    a.qh = s[2];
    a.dtype = dtype;
    a.out = out;
    a.part = static_cast<float*>(workspace);
    a.sinks = sinks;
    a.heads = heads;
    a.group = heads / a.c.kv_heads;
    a.seq = seq;
    a.rows = seq * a.group;
    a.window = window;
    a.splits = plan.splits;
    a.by_length = plan.by_length;
    a.scale2 = scale * 1.4426950408889634f;
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
