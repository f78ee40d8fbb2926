// Beam search: the best continuations over a sequence's beams and the vocabulary, and the states that follow them.
//
// Within a row (one beam) the order of the candidates is that of the logits, so a slice of a row is reduced to its `count` best logits
// and its share of the row's log-sum-exp in one pass; a second kernel, a CTA per group of beams, adds up the shares, gives the few
// candidates that are left their values in 64 bits (candidates of different beams lie close to one another, and float32 scores of
// long texts have steps of 1e-6 and more) and takes the best.
//
// Both find the best the same way.  Threads keep the largest of what they have seen; a bar that at least `count` threads reach, and not
// many more, is searched for by halving (about ten counts over the CTA); only what the threads that reach it have seen can be among the
// best, and is looked at again (a slice: from L2); what reaches the bar (a few dozen) is listed in shared memory, and each of those counts
// how many are better.  Where too many reach every bar (equal logits in thousands) the best are taken one by one.
#include "decoder.cuh"
#include "cache4.cuh"

namespace rb {

constexpr int BEAM_WIDTH = 32, BEAM_COUNT = 64;
constexpr int BEAM_THREADS = 512, BEAM_PIECE = 8;        // neighbouring logits that a thread takes at a time
constexpr int BEAM_ROUND = BEAM_THREADS * BEAM_PIECE;    // slices are whole rounds of a CTA
constexpr int BEAM_LIST = 1024;       // candidates that can be listed
constexpr uint32_t BEAM_NONE = 0x007fffffu;  // keys of candidates are above this, the key of -inf

// Unsigned numbers in the order of the floats.
__device__ __forceinline__ uint32_t order_key(float x) {
    x += 0.f;  // (-0 and 0 are equal)
    const uint32_t u = __float_as_uint(x);
    return x != x ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ unsigned long long order_key(double x) {
    x += 0.0;
    const unsigned long long u = (unsigned long long)__double_as_longlong(x);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

// Largest bar found by halving that at least `want` threads' `mine` reach, not above what few enough of them reach; at least `least`.
__device__ __forceinline__ uint32_t find_bar(uint32_t mine, uint32_t least, uint32_t top, int want) {
    uint32_t lo = least, hi = top;  // (at `lo` the count is enough, or nothing better is known)
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        const int n = __syncthreads_count(mine >= mid);
        if (n >= want)
            lo = mid;
        else
            hi = mid - 1;
        if (n >= want && n <= 2 * want) break;
    }
    return lo;
}

struct BeamSelect {
    const void* logits;
    size_t group_stride, beam_stride;
    int wide;
    const float* scores;
    const uint8_t* ended;
    int groups, width, vocab, count, slices, rounds;
    long long pad;
    float2* share;        // [rows][slices]: largest logit, sum of exp(logit - largest)
    uint2* list;          // [rows][slices][count]: key of the logit, token; keys BEAM_NONE and below are no candidates
    float* out_scores;
    long long *out_beams, *out_tokens;
};

// Logits i .. i + 7 of a row; what is no candidate as -inf.
template <typename T>
__device__ __forceinline__ void beam_piece(const T* x, int i, int vocab, int wide, float (&v)[BEAM_PIECE]) {
    if (i + BEAM_PIECE <= vocab) {
        load8(x + i, wide, v);
#pragma unroll
        for (int n = 0; n < BEAM_PIECE; ++n) v[n] = fmaxf(v[n], -INFINITY);  // (NaN: -inf)
    } else {
#pragma unroll
        for (int n = 0; n < BEAM_PIECE; ++n) v[n] = i + n < vocab ? fmaxf(type_load(x + i + n), -INFINITY) : -INFINITY;
    }
}

template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS) beam_slice_kernel(const __grid_constant__ BeamSelect p) {
    __shared__ float s_red[64];
    __shared__ uint2 s_list[BEAM_LIST];
    __shared__ unsigned short s_who[BEAM_THREADS];
    __shared__ int s_n, s_whos;
    __shared__ unsigned long long s_best;
    pdl_wait();
    pdl_trigger();
    const int row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x;
    if (p.ended && p.ended[row]) return;  // (the second kernel does not look at this row's share)
    const int group = row / p.width;
    const T* x = static_cast<const T*>(p.logits) + (size_t)group * p.group_stride + (size_t)(row - group * p.width) * p.beam_stride;
    const int base = slice * p.rounds * BEAM_ROUND, rounds = min(p.rounds, (p.vocab - base + BEAM_ROUND - 1) / BEAM_ROUND);
    auto place = [&](int round, int who) { return base + (round * BEAM_THREADS + who) * BEAM_PIECE; };

    // ---- largest logit and sum of exp(logit - largest) of this thread's pieces
    constexpr float log2e = 1.4426950408889634f;
    float largest = -INFINITY, sum = 0.f;
    auto take = [&](const float (&v)[BEAM_PIECE]) {
        float m = v[0];
#pragma unroll
        for (int n = 1; n < BEAM_PIECE; ++n) m = fmaxf(m, v[n]);
        if (m > largest) {
            sum *= fast_exp2((largest - m) * log2e);
            largest = m;
        }
        // (the difference first: the lowest float times log2(e) is none)
        const float off = largest == -INFINITY ? 0.f : largest;
#pragma unroll
        for (int n = 0; n < BEAM_PIECE; ++n) sum += fast_exp2((v[n] - off) * log2e);
    };
    int r = 0;
    for (; r + 4 <= rounds; r += 4) {
        float v[4][BEAM_PIECE];
#pragma unroll
        for (int k = 0; k < 4; ++k) beam_piece(x, place(r + k, tid), p.vocab, p.wide, v[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k) take(v[k]);
    }
    for (; r < rounds; ++r) {
        float v[BEAM_PIECE];
        beam_piece(x, place(r, tid), p.vocab, p.wide, v);
        take(v);
    }

    // ---- share of the row's mass
    const uint32_t mine = order_key(largest);
    const uint32_t top_key = __reduce_max_sync(0xffffffffu, mine);
    if ((tid & 31) == 0) reinterpret_cast<uint32_t*>(s_red)[tid >> 5] = top_key;
    if (tid == 0) s_n = s_whos = 0;
    __syncthreads();
    const uint32_t top = __reduce_max_sync(0xffffffffu, reinterpret_cast<uint32_t*>(s_red)[tid & (BEAM_THREADS / 32 - 1)]);
    const float most = order_value(top);
    sum = block_sum(largest == -INFINITY ? 0.f : sum * fast_exp2((largest - most) * log2e), s_red + 16);
    const size_t at = (size_t)row * p.slices + slice;
    if (tid == 0) p.share[at] = make_float2(most, sum);
    uint2* out = p.list + at * p.count;

    // ---- the best of the slice
    const uint32_t bar = find_bar(mine, BEAM_NONE + 1, top, p.count);
    if (mine >= bar && mine > BEAM_NONE) s_who[atomicAdd(&s_whos, 1)] = (unsigned short)tid;
    __syncthreads();
    const int pieces = s_whos * rounds;
    for (int i = tid; i < pieces; i += BEAM_THREADS) {
        const int who = i / rounds, at0 = place(i - who * rounds, s_who[who]);
        float v[BEAM_PIECE];
        beam_piece(x, at0, p.vocab, p.wide, v);
#pragma unroll
        for (int n = 0; n < BEAM_PIECE; ++n) {
            const uint32_t key = order_key(v[n]);
            if (key >= bar && key > BEAM_NONE) {
                const int k = atomicAdd(&s_n, 1);
                if (k < BEAM_LIST) s_list[k] = make_uint2(key, at0 + n);
            }
        }
    }
    __syncthreads();
    const int n = s_n;
    if (n <= BEAM_LIST) {
        for (int i = tid; i < n; i += BEAM_THREADS) {
            const uint2 c = s_list[i];
            int better = 0;
            for (int k = 0; k < n; ++k) {
                const uint2 d = s_list[k];
                better += d.x > c.x || (d.x == c.x && d.y < c.y);
            }
            if (better < p.count) out[better] = c;
        }
        for (int i = n + tid; i < p.count; i += BEAM_THREADS) out[i] = make_uint2(0u, 0u);
        return;
    }
    // too many that are equal: one by one, the largest key and among equals the lowest token, below the last one taken
    unsigned long long last = ~0ull;
    for (int k = 0; k < p.count; ++k) {
        unsigned long long best = 0;
        for (int i = 0; i < rounds; ++i) {
            float v[BEAM_PIECE];
            beam_piece(x, place(i, tid), p.vocab, p.wide, v);
#pragma unroll
            for (int m = 0; m < BEAM_PIECE; ++m) {
                const uint32_t key = order_key(v[m]);
                const unsigned long long c = (unsigned long long)key << 32 | ~(uint32_t)(place(i, tid) + m);
                if (key > BEAM_NONE && c < last && c > best) best = c;
            }
        }
        if (tid == 0) s_best = 0;
        __syncthreads();
        atomicMax(&s_best, best);
        __syncthreads();
        last = s_best;
        __syncthreads();
        if (tid == 0) out[k] = last ? make_uint2((uint32_t)(last >> 32), ~(uint32_t)last) : make_uint2(0u, 0u);
    }
}

struct Candidate {
    unsigned long long key;  // of the value in 64 bits
    uint32_t flat;           // beam * vocab + token
};
__device__ __forceinline__ bool better_than(const Candidate& a, const Candidate& b) {
    return a.key > b.key || (a.key == b.key && a.flat < b.flat);
}
__device__ __forceinline__ double candidate_value(unsigned long long key) {
    return __longlong_as_double((long long)(key >> 63 ? key & 0x7fffffffffffffffull : ~key));
}

__global__ void __launch_bounds__(BEAM_THREADS) beam_join_kernel(const __grid_constant__ BeamSelect p) {
    __shared__ double s_base[BEAM_WIDTH], s_lse[BEAM_WIDTH];
    __shared__ int s_kind[BEAM_WIDTH];  // 0: offers nothing, 1: goes on, 2: ended
    __shared__ Candidate s_list[BEAM_LIST], s_out[BEAM_COUNT];
    __shared__ uint32_t s_top[BEAM_THREADS / 32];
    __shared__ int s_n;
    __shared__ Candidate s_best;
    pdl_wait();
    pdl_trigger();
    const int group = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int w = warp; w < p.width; w += BEAM_THREADS / 32) {
        const int row = group * p.width + w;
        const float score = p.scores[row];
        const bool ended = p.ended && p.ended[row];
        double lse = 0.0;
        bool fine = isfinite(score);
        if (!ended) {
            float top = -INFINITY;
            for (int s = lane; s < p.slices; s += 32) top = fmaxf(top, __ldcg(&p.share[(size_t)row * p.slices + s]).x);
            top = warp_max(top);
            double sum = 0.0;
            for (int s = lane; s < p.slices; s += 32) {
                const float2 v = __ldcg(&p.share[(size_t)row * p.slices + s]);
                if (v.x != -INFINITY) sum += (double)v.y * exp((double)v.x - (double)top);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            fine = fine && isfinite(top);
            lse = (double)top + log(sum);
        }
        if (lane == 0) {
            s_kind[w] = !fine ? 0 : ended ? 2 : 1;
            s_base[w] = (double)score;
            s_lse[w] = lse;
        }
    }
    if (tid == 0) s_n = 0;
    __syncthreads();

    const int per_row = p.slices * p.count, n_all = p.width * per_row;
    // candidate i of the lists; an ended beam's one stands in its first place
    auto candidate = [&](int i) {
        const int w = i / per_row;
        Candidate c = {0ull, 0u};
        if (s_kind[w] == 2) {
            if (i == w * per_row) c = Candidate{order_key(s_base[w]), (uint32_t)((size_t)w * p.vocab + p.pad)};
        } else if (s_kind[w] == 1) {
            const uint2 l = __ldcg(&p.list[(size_t)group * n_all + i]);
            if (l.x > BEAM_NONE)
                c = Candidate{order_key(s_base[w] + ((double)order_value(l.x) - s_lse[w])), (uint32_t)((size_t)w * p.vocab + l.y)};
        }
        return c;
    };
    uint32_t mine = 0;
    for (int i = tid; i < n_all; i += BEAM_THREADS) mine = max(mine, (uint32_t)(candidate(i).key >> 32));
    const uint32_t wtop = __reduce_max_sync(0xffffffffu, mine);
    if (lane == 0) s_top[warp] = wtop;
    __syncthreads();
    const uint32_t top = __reduce_max_sync(0xffffffffu, s_top[lane & (BEAM_THREADS / 32 - 1)]);
    const uint32_t bar = find_bar(mine, 1u, max(top, 1u), p.count);
    for (int i = tid; i < n_all; i += BEAM_THREADS) {
        const Candidate c = candidate(i);
        if (c.key && (uint32_t)(c.key >> 32) >= bar) {
            const int n = atomicAdd(&s_n, 1);
            if (n < BEAM_LIST) s_list[n] = c;
        }
    }
    __syncthreads();
    const int n = s_n;
    int found = min(n, p.count);
    if (n <= BEAM_LIST) {
        for (int i = tid; i < n; i += BEAM_THREADS) {
            const Candidate c = s_list[i];
            int better = 0;
            for (int k = 0; k < n; ++k) better += better_than(s_list[k], c);
            if (better < p.count) s_out[better] = c;
        }
    } else {  // one by one: the best that is worse than the last one taken
        Candidate last = {~0ull, 0u};
        for (int k = 0; k < p.count; ++k) {
            Candidate best = {0ull, 0u};
            for (int i = tid; i < n_all; i += BEAM_THREADS) {
                const Candidate c = candidate(i);
                if (c.key && better_than(last, c) && better_than(c, best)) best = c;
            }
            for (int o = 16; o > 0; o >>= 1) {
                Candidate c;
                c.key = __shfl_xor_sync(0xffffffffu, best.key, o);
                c.flat = __shfl_xor_sync(0xffffffffu, best.flat, o);
                if (better_than(c, best)) best = c;
            }
            __syncthreads();
            if (lane == 0) s_list[warp] = best;
            __syncthreads();
            if (tid == 0) {
                for (int w = 1; w < BEAM_THREADS / 32; ++w)
                    if (better_than(s_list[w], best)) best = s_list[w];
                s_out[k] = s_best = best;
            }
            __syncthreads();
            last = s_best;
        }
    }
    __syncthreads();
    // fewer candidates than asked for: -inf and the lowest places that are not among them
    if (tid == 0 && found < p.count) {
        const int real = found;
        for (uint32_t flat = 0; found < p.count; ++flat) {
            bool taken = false;
            for (int k = 0; k < real; ++k) taken |= s_out[k].flat == flat;
            if (!taken) s_out[found++] = Candidate{0ull, flat};
        }
    }
    __syncthreads();
    if (tid < p.count) {
        const Candidate c = s_out[tid];
        const size_t at = (size_t)group * p.count + tid;
        p.out_scores[at] = c.key ? (float)candidate_value(c.key) : -INFINITY;
        p.out_beams[at] = c.flat / (uint32_t)p.vocab;
        p.out_tokens[at] = c.flat % (uint32_t)p.vocab;
    }
}

// ---------------------------------------------------------------- states
// A thread owns one piece of up to 16 bytes of every row of a group: it reads what the moving rows take from the others, then writes, so
// the rows change places in place, each byte that moves is read and written once, and no thread waits for another.
constexpr int REORDER_STATES = 64, REORDER_THREADS = 256;

struct ReorderState {
    unsigned char* data;
    size_t row_stride, segment_stride;
    uint32_t units;      // pieces of a row
    uint32_t first;      // CTA (of the launch's x) that its pieces begin at
    FastDiv per_segment;
    int unit;            // bytes of a piece: 16, 8, 4, 2 or 1
};
struct Reorder {
    ReorderState s[REORDER_STATES];
    int n, width;
    const long long* beams;
};

template <int W, typename T>
__device__ __forceinline__ void move_rows(unsigned char* at, size_t stride, const int* source, int width) {
    T v[W];
#pragma unroll
    for (int w = 0; w < W; ++w)
        if (w < width && source[w] != w) v[w] = *reinterpret_cast<const T*>(at + source[w] * stride);
#pragma unroll
    for (int w = 0; w < W; ++w)
        if (w < width && source[w] != w) *reinterpret_cast<T*>(at + w * stride) = v[w];
}

template <int W>
__global__ void __launch_bounds__(REORDER_THREADS) reorder_kernel(const __grid_constant__ Reorder p) {
    __shared__ int s_source[W];
    pdl_wait();
    pdl_trigger();
    if (threadIdx.x < p.width) {
        const long long w = p.beams[(size_t)blockIdx.y * p.width + threadIdx.x];
        s_source[threadIdx.x] = w >= 0 && w < p.width ? (int)w : threadIdx.x;
    }
    __syncthreads();
    int k = 0;
    while (k + 1 < p.n && p.s[k + 1].first <= blockIdx.x) ++k;
    const ReorderState& s = p.s[k];
    const uint32_t u = (blockIdx.x - s.first) * REORDER_THREADS + threadIdx.x;
    if (u >= s.units) return;
    const uint32_t segment = s.per_segment.div(u), piece = u - segment * s.per_segment.d;
    unsigned char* at = s.data + (size_t)blockIdx.y * p.width * s.row_stride + segment * s.segment_stride + (size_t)piece * s.unit;
    switch (s.unit) {
        case 16: move_rows<W, uint4>(at, s.row_stride, s_source, p.width); break;
        case 8: move_rows<W, uint2>(at, s.row_stride, s_source, p.width); break;
        case 4: move_rows<W, uint32_t>(at, s.row_stride, s_source, p.width); break;
        case 2: move_rows<W, uint16_t>(at, s.row_stride, s_source, p.width); break;
        default: move_rows<W, uint8_t>(at, s.row_stride, s_source, p.width); break;
    }
}

// Rounds of a slice: as few as keep two CTAs on every SM busy, so that a slice's fixed part (the bar, the list) is shared by what it can be.
static int beam_rounds(int rows, int vocab) {
    const int all = (vocab + BEAM_ROUND - 1) / BEAM_ROUND;
    const int slices = (2 * fused_sm_count() + rows - 1) / rows;
    return slices >= all ? 1 : (all + slices - 1) / slices;
}
static int beam_slices(int rows, int vocab) {
    const int per = beam_rounds(rows, vocab) * BEAM_ROUND;
    return (vocab + per - 1) / per;
}
static bool beam_shape(int groups, int width, int vocab, int count) {
    return groups > 0 && width > 0 && vocab > 0 && count > 0 && width <= BEAM_WIDTH && count <= BEAM_COUNT &&
           vocab <= (1 << 30) && (long long)width * vocab < (1LL << 31) && count <= (long long)width * vocab && (long long)groups * width <= 65535;
}

}  // namespace rb

using namespace rb;

extern "C" {

size_t rotor_b200_beam_select_workspace_bytes(int groups, int width, int vocab, int count) {
    if (!beam_shape(groups, width, vocab, count)) return 0;
    return (size_t)groups * width * beam_slices(groups * width, vocab) * (sizeof(float2) + count * sizeof(uint2));
}

int rotor_b200_beam_select(const void* logits, int dtype, int64_t group_stride, int64_t beam_stride, const float* scores,
                           const uint8_t* ended, int groups, int width, int vocab, int count, int64_t pad, float* out_scores,
                           int64_t* out_beams, int64_t* out_tokens, void* workspace, size_t workspace_bytes, void* stream) {
    RB_REQUIRE(logits && scores && out_scores && out_beams && out_tokens && workspace && ((uintptr_t)workspace & 15) == 0);
    RB_REQUIRE(dtype >= ROTOR_B200_F32 && dtype <= ROTOR_B200_F16 && group_stride >= 0 && beam_stride >= 0);
    RB_REQUIRE(!ended || (pad >= 0 && pad < vocab));
    if (!beam_shape(groups, width, vocab, count)) return ROTOR_B200_ERR_SHAPE;
    if (workspace_bytes < rotor_b200_beam_select_workspace_bytes(groups, width, vocab, count)) return ROTOR_B200_ERR_WORKSPACE;
    const int size = dtype == ROTOR_B200_F32 ? 4 : 2;
    RB_REQUIRE((uintptr_t)logits % size == 0);
    BeamSelect p;
    p.logits = logits;
    p.group_stride = group_stride;
    p.beam_stride = beam_stride;
    p.wide = (((uintptr_t)logits | (uintptr_t)((group_stride | beam_stride) * size)) & 15) == 0;
    p.scores = scores;
    p.ended = ended;
    p.groups = groups;
    p.width = width;
    p.vocab = vocab;
    p.count = count;
    p.slices = beam_slices(groups * width, vocab);
    p.rounds = beam_rounds(groups * width, vocab);
    p.pad = ended ? pad : 0;
    const size_t shares = (size_t)groups * width * p.slices;
    p.list = static_cast<uint2*>(workspace);
    p.share = reinterpret_cast<float2*>(p.list + shares * count);
    p.out_scores = out_scores;
    p.out_beams = reinterpret_cast<long long*>(out_beams);
    p.out_tokens = reinterpret_cast<long long*>(out_tokens);
    const cudaStream_t st = as_stream(stream);
    const dim3 grid(p.slices, groups * width);
    int e;
    switch (dtype) {
        case ROTOR_B200_F32: e = launch_chained(beam_slice_kernel<float>, grid, BEAM_THREADS, 0, st, 1, p); break;
        case ROTOR_B200_BF16: e = launch_chained(beam_slice_kernel<__nv_bfloat16>, grid, BEAM_THREADS, 0, st, 1, p); break;
        default: e = launch_chained(beam_slice_kernel<__half>, grid, BEAM_THREADS, 0, st, 1, p); break;
    }
    return e ? e : launch_chained(beam_join_kernel, dim3(groups), BEAM_THREADS, 0, st, 1, p);
}

int rotor_b200_reorder_states(const rotor_b200_state* states, int n, const int64_t* beams, int groups, int width, void* stream) {
    RB_REQUIRE(states && beams && n > 0 && groups > 0 && width > 0);
    if (width > BEAM_WIDTH || groups > 65535) return ROTOR_B200_ERR_SHAPE;
    for (int i = 0; i < n; ++i) {
        const rotor_b200_state& s = states[i];
        RB_REQUIRE(s.data && s.segments > 0);
        RB_REQUIRE(s.segments == 1 || s.segment_stride >= s.segment_bytes);
        for (int k = 0; k < i; ++k) RB_REQUIRE(states[k].data != s.data);  // (moved twice, by threads that do not wait for one another)
        RB_REQUIRE(groups * width == 1 || s.row_stride >= (size_t)(s.segments - 1) * s.segment_stride + s.segment_bytes);
    }
    const cudaStream_t st = as_stream(stream);
    for (int begin = 0; begin < n;) {
        Reorder p;
        p.n = 0;
        p.width = width;
        p.beams = reinterpret_cast<const long long*>(beams);
        uint64_t blocks = 0;
        for (; begin < n && p.n < REORDER_STATES; ++begin) {
            const rotor_b200_state& s = states[begin];
            if (s.segment_bytes == 0) continue;
            const uintptr_t all = (uintptr_t)s.data | s.row_stride | (s.segments > 1 ? s.segment_stride : 0) | s.segment_bytes;
            int unit = 16;
            while (all & (unit - 1)) unit >>= 1;
            const uint64_t per = s.segment_bytes / unit, units = per * s.segments;
            if (units > 0x7fffff00u) return ROTOR_B200_ERR_SHAPE;
            const uint64_t more = (units + REORDER_THREADS - 1) / REORDER_THREADS;
            if (blocks + more > 0x7fffffffu) break;
            ReorderState& d = p.s[p.n++];
            d.data = static_cast<unsigned char*>(s.data);
            d.row_stride = s.row_stride;
            d.segment_stride = s.segment_stride;
            d.units = (uint32_t)units;
            d.first = (uint32_t)blocks;
            d.per_segment = FastDiv((uint32_t)per);
            d.unit = unit;
            blocks += more;
        }
        if (!p.n) break;
        const dim3 grid((unsigned)blocks, groups);
        int e;
        if (width <= 4)
            e = launch_chained(reorder_kernel<4>, grid, REORDER_THREADS, 0, st, 1, p);
        else if (width <= 8)
            e = launch_chained(reorder_kernel<8>, grid, REORDER_THREADS, 0, st, 1, p);
        else if (width <= 16)
            e = launch_chained(reorder_kernel<16>, grid, REORDER_THREADS, 0, st, 1, p);
        else
            e = launch_chained(reorder_kernel<32>, grid, REORDER_THREADS, 0, st, 1, p);
        if (e) return e;
    }
    return ROTOR_B200_OK;
}

}  // extern "C"
