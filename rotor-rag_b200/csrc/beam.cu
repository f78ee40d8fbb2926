// Beam search: the best continuations over a sequence's beams and the vocabulary, and the states that follow them.
//
// Within a row (one beam) the order of the candidates is that of the logits, so a CTA reduces its part of a row to the `count` best logits
// and its share of the row's log-sum-exp in one pass; then one CTA per group of beams adds up the shares, gives the few candidates that are
// left their values in 64 bits (float32 scores of long texts have steps of 1e-6 and more, in which candidates of different beams would be
// equal) and takes the best.  The sum itself is float32, off by 2e-7 where the most was measured: in 64 bits an exponential of a polynomial
// would be some 15 instructions a logit, by the rate of double precision an estimated 14 us for 128 rows of 128256.  Two forms: a group's CTAs are a cluster, whose first one reads the others' shared memory (one launch, no
// workspace), or the parts are a launch of their own that fills the GPU, and their offers pass through a workspace.  4 beams of 102400
// logits: 10.8 us as a cluster, 8.2 as two launches, of which the second costs the host 3 us and more; 128 beams of 128256: 33 / 20.
//
// Both stages find the best the same way.  Threads keep the largest of what they have seen; a bar that at least `count` threads reach, and
// too many more, comes from the warps' largest, and is raised by halving where that is not enough; only what the threads that reach it have
// seen can be among the best, and is looked at again (logits: from L2); what reaches the bar (a few dozen) is listed in shared memory, where
// eight threads count for each how many are better.  Where too many reach every bar (equal logits in thousands) the best are taken one by
// one.
#include "decoder.cuh"
#include "cache4.cuh"

namespace rb {

constexpr int BEAM_WIDTH = 32, BEAM_COUNT = 64;
constexpr int BEAM_CLUSTER = 16;                         // most CTAs of a group (more than 8 where the device can place them)
constexpr int BEAM_ROWS = BEAM_WIDTH / 8;                // most rows of a CTA
constexpr int BEAM_THREADS = 512, BEAM_PIECE = 8;        // neighbouring logits that a thread takes at a time
constexpr int BEAM_ROUND = BEAM_THREADS * BEAM_PIECE;    // slices are whole rounds of a CTA
constexpr int BEAM_DEPTH = 4;         // rounds of a CTA's ring
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

// A bar that at least `want` threads' `mine` reach (or all, where fewer are above `least`), and, but for equal ones, not many more.  Of
// `want` sets of threads each has one that reaches the smallest of the sets' largest, which is where the search between that and the largest
// of all begins (for random numbers and up to sixteen sets, the warps, it ends there).  s_sets: BEAM_COUNT words.
__device__ __forceinline__ uint32_t find_bar(uint32_t mine, uint32_t least, int want, uint32_t* s_sets, uint32_t& top) {
    const int lane = threadIdx.x & 31, set_lanes = want <= BEAM_THREADS / 32 ? 32 : want <= BEAM_THREADS / 16 ? 16 : 8;
    uint32_t most = mine;
    for (int o = 1; o < set_lanes; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    if ((threadIdx.x & (set_lanes - 1)) == 0) s_sets[threadIdx.x / set_lanes] = most;
    __syncthreads();
    const int sets = BEAM_THREADS / set_lanes;  // 16, 32 or 64
    const uint32_t a = s_sets[lane & (sets - 1)], b = s_sets[(lane + 32) & (sets - 1)];
    top = __reduce_max_sync(0xffffffffu, max(a, b));
    uint32_t lo = max(__reduce_min_sync(0xffffffffu, min(a, b)), least), hi = top;
    int n = __syncthreads_count(mine >= lo);
    const int few = max(48, 2 * want);
    while (lo < hi && n > few) {  // (at `lo` the count is enough, or nothing better is known)
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        const int k = __syncthreads_count(mine >= mid);
        if (k >= want) {
            lo = mid;
            n = k;
        } else {
            hi = mid - 1;
        }
    }
    return lo;
}

// The first of `count` places behind those taken of a list: one addition per warp (additions to one word are done one by one).
__device__ __forceinline__ int take_places(int count, int* taken) {
    const int lane = threadIdx.x & 31;
    int upto = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int below = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += below;
    }
    int base = 0;
    if (lane == 31 && upto) base = atomicAdd(taken, upto);
    return __shfl_sync(0xffffffffu, base, 31) + upto - count;
}

// How many of n listed ones are better than number i: by eight neighbouring threads, `sub` of which this is.
template <typename Better>
__device__ __forceinline__ int count_better(int n, int sub, Better better) {
    int count = 0;
    for (int k = sub; k < n; k += 8) count += better(k);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) count += __shfl_xor_sync(0xffffffffu, count, o);
    return count;
}

struct BeamSelect {
    const void* logits;
    size_t group_stride, beam_stride;
    int wide;
    const float* scores;
    const uint8_t* ended;
    int groups, width, vocab, count;
    int cluster;                 // CTAs of a group; 0: two launches
    int parts, rounds;           // CTAs that share a row (a cluster's CTA may take several rows), rounds of a CTA's part
    long long pad;
    FastDiv per_row;             // candidates of a row: parts * count
    float2* share;               // two launches: [row][part]: largest logit, sum of exp(logit - largest)
    uint2* list;                 // [row][part][count]: key and token
    float* out_scores;
    long long *out_beams, *out_tokens;
};

// A thread's eight logits of a round, 16 bytes at a time (so a warp's loads are whole lines): place n of thread `who`.
template <typename T>
__device__ __forceinline__ int beam_place(int begin, int who, int n) {
    return sizeof(T) == 4 ? begin + n / 4 * (BEAM_ROUND / 2) + who * 4 + n % 4 : begin + who * 8 + n;
}
// ... what is no candidate as -inf.
template <typename T>
__device__ __forceinline__ void beam_piece(const T* x, int begin, int who, int vocab, int wide, float (&v)[BEAM_PIECE]) {
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int k = 0; k < BEAM_PIECE; k += N) {
        const int i = beam_place<T>(begin, who, k);
        if (wide && i + N <= vocab) {
            const uint4 w = *reinterpret_cast<const uint4*>(x + i);
            const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
            for (int n = 0; n < N; ++n) v[k + n] = type_load(t + n);
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n) v[k + n] = i + n < vocab ? type_load(x + i + n) : -INFINITY;
        }
    }
#pragma unroll
    for (int n = 0; n < BEAM_PIECE; ++n) v[n] = fmaxf(v[n], -INFINITY);  // (NaN: -inf)
}

// What a CTA hands to its cluster's first one.
struct BeamOffer {
    float2 share[BEAM_ROWS];            // of each row that it takes: largest logit, sum of exp(logit - largest)
    uint2 list[BEAM_ROWS][BEAM_COUNT];  // key and token; keys BEAM_NONE and below are no candidates
};
struct Candidate {
    unsigned long long key;  // of the value in 64 bits
    uint32_t flat;           // beam * vocab + token
};
struct BeamShared {
    union {
        uint2 list[BEAM_LIST];
        Candidate best[BEAM_LIST];
    };
    Candidate out[BEAM_COUNT], taken;
    double base[BEAM_WIDTH], lse[BEAM_WIDTH];
    int kind[BEAM_WIDTH];    // 0: offers nothing, 1: goes on, 2: ended
    float red[33];
    uint32_t sets[BEAM_COUNT];
    unsigned short who[BEAM_THREADS];
    int n, whos;
    unsigned long long top;
};

__device__ __forceinline__ bool better_than(const Candidate& a, const Candidate& b) {
    return a.key > b.key || (a.key == b.key && a.flat < b.flat);
}
__device__ __forceinline__ double candidate_value(unsigned long long key) {
    return __longlong_as_double((long long)(key >> 63 ? key & 0x7fffffffffffffffull : ~key));
}

// A row's part [base, base + rounds BEAM_ROUND): share and the best logits.
template <typename T>
__device__ void beam_part(const BeamSelect& p, const T* x, int base, BeamShared& sh, float2& share, uint2* out) {
    const int tid = threadIdx.x, rounds = min(p.rounds, (p.vocab - base + BEAM_ROUND - 1) / BEAM_ROUND);
    // ---- largest logit and sum of exp(logit - largest) of this thread's pieces
    constexpr float log2e = 1.4426950408889634f;
    float largest = -INFINITY, sum = 0.f, v[BEAM_PIECE];
    auto take = [&]() {  // (by pairs: the chain from one round to the next is short)
        float m[BEAM_PIECE / 2];
#pragma unroll
        for (int n = 0; n < BEAM_PIECE / 2; ++n) m[n] = fmaxf(v[2 * n], v[2 * n + 1]);  // (passes over NaN)
        const float most = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
        if (most > largest) {
            sum *= fast_exp2((largest - most) * log2e);
            largest = most;
        }
        // (the difference first: the lowest float times log2(e) is none)
        const float off = largest == -INFINITY ? 0.f : -largest;
        float2 e[BEAM_PIECE / 2];
#pragma unroll
        for (int n = 0; n < BEAM_PIECE / 2; ++n) {
            e[n] = __fmul2_rn(__fadd2_rn(make_float2(v[2 * n], v[2 * n + 1]), make_float2(off, off)), make_float2(log2e, log2e));
            e[n] = make_float2(fast_exp2(e[n].x), fast_exp2(e[n].y));
        }
        const float2 part = __fadd2_rn(__fadd2_rn(e[0], e[1]), __fadd2_rn(e[2], e[3]));
        sum += part.x + part.y;
    };
    // Whole rounds pass through a ring in shared memory, of which a thread copies and reads its own pieces: the loads in flight do not
    // depend on the registers, and nobody waits for another.
    extern __shared__ __align__(16) unsigned char beam_raw[];
    constexpr int N = 16 / sizeof(T), COPIES = BEAM_PIECE / N, BYTES = BEAM_ROUND * sizeof(T);
    const int whole = p.wide ? min(rounds, max(p.vocab - base, 0) / BEAM_ROUND) : 0;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(beam_raw) + tid * 16;
    const T* from = x + base + tid * N;
    auto fetch = [&](int r, int slot) {
        if (r < whole) {
#pragma unroll
            for (int k = 0; k < COPIES; ++k)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ring + slot * BYTES + k * BEAM_THREADS * 16),
                             "l"(from + (size_t)r * BEAM_ROUND + k * BEAM_THREADS * N)
                             : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int r = 0; r < BEAM_DEPTH - 1; ++r) fetch(r, r);
    for (int r = 0; r < whole; r += BEAM_DEPTH) {
#pragma unroll
        for (int k = 0; k < BEAM_DEPTH; ++k) {
            if (r + k < whole) {
                fetch(r + k + BEAM_DEPTH - 1, (k + BEAM_DEPTH - 1) % BEAM_DEPTH);
                asm volatile("cp.async.wait_group %0;" ::"n"(BEAM_DEPTH - 1) : "memory");
#pragma unroll
                for (int c = 0; c < COPIES; ++c) {
                    const uint4 w = *reinterpret_cast<const uint4*>(beam_raw + k * BYTES + (c * BEAM_THREADS + tid) * 16);
#pragma unroll
                    for (int n = 0; n < N; ++n) v[c * N + n] = type_load(reinterpret_cast<const T*>(&w) + n);
                }
                take();
            }
        }
    }
    for (int r = whole; r < rounds; ++r) {
        beam_piece(x, base + r * BEAM_ROUND, tid, p.vocab, p.wide, v);
        take();
    }
    if (sum != sum) {  // NaN among the logits: again, without it (and with +inf, which takes the row out)
        sum = 0.f;
        for (int r = 0; r < rounds; ++r) {
            beam_piece(x, base + r * BEAM_ROUND, tid, p.vocab, p.wide, v);
#pragma unroll
            for (int n = 0; n < BEAM_PIECE; ++n)
                if (v[n] > -INFINITY) sum += fast_exp2((v[n] - largest) * log2e);
        }
    }

    // ---- share of the row's mass
    const uint32_t mine = order_key(largest);
    uint32_t top;
    if (tid == 0) sh.n = sh.whos = 0;
    const uint32_t bar = find_bar(mine, BEAM_NONE + 1, p.count, sh.sets, top);
    const float most = order_value(top);
    sum = block_sum(largest == -INFINITY ? 0.f : sum * fast_exp2((largest - most) * log2e), sh.red);
    if (tid == 0) share = make_float2(most, sum);

    // ---- the best of the part
    const bool reaches = mine >= bar && mine > BEAM_NONE;
    const int mark = take_places(reaches, &sh.whos);
    if (reaches) sh.who[mark] = (unsigned short)tid;
    __syncthreads();
    const int pieces = sh.whos * rounds;
    for (int i0 = 0; i0 < pieces; i0 += BEAM_THREADS) {
        const int i = i0 + tid, k = i / rounds, who = sh.who[i < pieces ? k : 0], begin = base + (i - k * rounds) * BEAM_ROUND;
        int hits = 0;
        if (i < pieces) {
            beam_piece(x, begin, who, p.vocab, p.wide, v);
#pragma unroll
            for (int n = 0; n < BEAM_PIECE; ++n) {
                const uint32_t key = order_key(v[n]);
                hits |= (key >= bar && key > BEAM_NONE) << n;
            }
        }
        int at = take_places(__popc(hits), &sh.n);
#pragma unroll
        for (int n = 0; n < BEAM_PIECE; ++n) {
            if (hits >> n & 1) {
                if (at < BEAM_LIST) sh.list[at] = make_uint2(order_key(v[n]), beam_place<T>(begin, who, n));
                ++at;
            }
        }
    }
    __syncthreads();
    const int n = sh.n;
    if (n <= BEAM_LIST) {
        for (int i0 = 0; i0 < n; i0 += BEAM_THREADS / 8) {
            const int i = i0 + tid / 8;
            const uint2 c = sh.list[min(i, n - 1)];
            const int better = count_better(n, tid & 7, [&](int k) {
                const uint2 d = sh.list[k];
                return d.x > c.x || (d.x == c.x && d.y < c.y);
            });
            if ((tid & 7) == 0 && i < n && better < p.count) out[better] = c;
        }
        for (int i = n + tid; i < p.count; i += BEAM_THREADS) out[i] = make_uint2(0u, 0u);
        __syncthreads();  // (the lists are used again)
        return;
    }
    // too many that are equal: one by one, the largest key and among equals the lowest token, below the last one taken
    unsigned long long last = ~0ull;
    for (int k = 0; k < p.count; ++k) {
        unsigned long long best = 0;
        for (int i = 0; i < rounds; ++i) {
            const int begin = base + i * BEAM_ROUND;
            beam_piece(x, begin, tid, p.vocab, p.wide, v);
#pragma unroll
            for (int m = 0; m < BEAM_PIECE; ++m) {
                const uint32_t key = order_key(v[m]);
                const unsigned long long c = (unsigned long long)key << 32 | ~(uint32_t)beam_place<T>(begin, tid, m);
                if (key > BEAM_NONE && c < last && c > best) best = c;
            }
        }
        if (tid == 0) sh.top = 0;
        __syncthreads();
        atomicMax(&sh.top, best);
        __syncthreads();
        last = sh.top;
        __syncthreads();
        if (tid == 0) out[k] = last ? make_uint2((uint32_t)(last >> 32), ~(uint32_t)last) : make_uint2(0u, 0u);
    }
}

// The best of a group: share_of(row, part) and offer_of(row, part, place) are what the parts left (at most 32 parts a row).
template <typename Share, typename Offer>
__device__ void beam_final(const BeamSelect& p, int group, BeamShared& sh, Share share_of, Offer offer_of) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per_row = p.parts * p.count, n_all = p.width * per_row;
    for (int w = warp; w < p.width; w += BEAM_THREADS / 32) {
        const int row = group * p.width + w;
        const float score = p.scores[row];
        const bool ended = p.ended && p.ended[row];
        double lse = 0.0;
        bool fine = isfinite(score);
        if (!ended) {
            const float2 v = lane < p.parts ? share_of(w, lane) : make_float2(-INFINITY, 0.f);
            const float top = warp_max(v.x);
            double sum = v.x != -INFINITY ? (double)(v.y * expf(v.x - top)) : 0.0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            fine = fine && isfinite(top);
            lse = (double)top + log(sum);
        }
        if (lane == 0) {
            sh.kind[w] = !fine ? 0 : ended ? 2 : 1;
            sh.base[w] = (double)score;
            sh.lse[w] = lse;
        }
    }
    if (tid == 0) sh.n = 0;
    __syncthreads();
    // candidate i: place i % count of a list; an ended beam's one stands in its first place
    auto candidate = [&](int i) {
        const int w = p.per_row.div(i), in_row = i - w * per_row;
        Candidate c = {0ull, 0u};
        if (sh.kind[w] == 2) {
            if (in_row == 0) c = Candidate{order_key(sh.base[w]), (uint32_t)((size_t)w * p.vocab + p.pad)};
        } else if (sh.kind[w] == 1) {
            const int k = in_row / p.count;
            const uint2 l = offer_of(w, k, in_row - k * p.count);
            if (l.x > BEAM_NONE)
                c = Candidate{order_key(sh.base[w] + ((double)order_value(l.x) - sh.lse[w])), (uint32_t)((size_t)w * p.vocab + l.y)};
        }
        return c;
    };
    constexpr int KEPT = 2;  // a thread's first candidates stay in registers
    Candidate own[KEPT];
    uint32_t mine = 0;
#pragma unroll
    for (int k = 0; k < KEPT; ++k) {
        const int i = tid + k * BEAM_THREADS;
        own[k] = i < n_all ? candidate(i) : Candidate{0ull, 0u};
        mine = max(mine, (uint32_t)(own[k].key >> 32));
    }
    for (int i = tid + KEPT * BEAM_THREADS; i < n_all; i += BEAM_THREADS) mine = max(mine, (uint32_t)(candidate(i).key >> 32));
    uint32_t top;
    const uint32_t bar = find_bar(mine, 1u, p.count, sh.sets, top);
    auto list = [&](const Candidate& c) {
        const bool reaches = c.key && (uint32_t)(c.key >> 32) >= bar;
        const int at = take_places(reaches, &sh.n);
        if (reaches && at < BEAM_LIST) sh.best[at] = c;
    };
#pragma unroll
    for (int k = 0; k < KEPT; ++k) list(own[k]);
    for (int i0 = KEPT * BEAM_THREADS; i0 < n_all; i0 += BEAM_THREADS) list(i0 + tid < n_all ? candidate(i0 + tid) : Candidate{0ull, 0u});
    __syncthreads();
    const int n = sh.n;
    int found = min(n, p.count);
    if (n <= BEAM_LIST) {
        for (int i0 = 0; i0 < n; i0 += BEAM_THREADS / 8) {
            const int i = i0 + tid / 8;
            const Candidate c = sh.best[min(i, n - 1)];
            const int better = count_better(n, tid & 7, [&](int k) { return better_than(sh.best[k], c); });
            if ((tid & 7) == 0 && i < n && better < p.count) sh.out[better] = c;
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
            if (lane == 0) sh.best[warp] = best;
            __syncthreads();
            if (tid == 0) {
                for (int w = 1; w < BEAM_THREADS / 32; ++w)
                    if (better_than(sh.best[w], best)) best = sh.best[w];
                sh.out[k] = sh.taken = best;
            }
            __syncthreads();
            last = sh.taken;
        }
    }
    __syncthreads();
    // fewer candidates than asked for: -inf and the lowest places that are not among them
    if (tid == 0 && found < p.count) {
        const int real = found;
        for (uint32_t flat = 0; found < p.count; ++flat) {
            bool taken = false;
            for (int k = 0; k < real; ++k) taken |= sh.out[k].flat == flat;
            if (!taken) sh.out[found++] = Candidate{0ull, flat};
        }
    }
    __syncthreads();
    if (tid < p.count) {
        const Candidate c = sh.out[tid];
        const size_t at = (size_t)group * p.count + tid;
        p.out_scores[at] = c.key ? (float)candidate_value(c.key) : -INFINITY;
        p.out_beams[at] = c.flat / (uint32_t)p.vocab;
        p.out_tokens[at] = c.flat % (uint32_t)p.vocab;
    }
}

template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS) beam_cluster_kernel(const __grid_constant__ BeamSelect p) {
    __shared__ BeamShared sh;
    __shared__ BeamOffer offer;
    pdl_wait();
    pdl_trigger();
    const int group = blockIdx.x / p.cluster, rank = blockIdx.x - group * p.cluster;
    const int w0 = rank / p.parts, part = rank - w0 * p.parts, step = p.cluster / p.parts;
    for (int w = w0, slot = 0; w < p.width; w += step, ++slot) {
        if (p.ended && p.ended[group * p.width + w]) continue;  // (nobody looks at its share)
        const T* x = static_cast<const T*>(p.logits) + (size_t)group * p.group_stride + (size_t)w * p.beam_stride;
        beam_part(p, x, part * p.rounds * BEAM_ROUND, sh, offer.share[slot], offer.list[slot]);
    }
    cluster_sync();
    if (rank == 0) {
        // part k of row w lies with CTA (w % step) parts + k, in its place w / step
        beam_final(
            p, group, sh, [&](int w, int k) { return cluster_load2(reinterpret_cast<const float*>(&offer.share[w / step]), w % step * p.parts + k); },
            [&](int w, int k, int i) {
                const float2 f = cluster_load2(reinterpret_cast<const float*>(&offer.list[w / step][i]), w % step * p.parts + k);
                return make_uint2(__float_as_uint(f.x), __float_as_uint(f.y));
            });
    }
    cluster_sync();  // (nobody leaves while its offers are being read)
}

template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS) beam_part_kernel(const __grid_constant__ BeamSelect p) {
    __shared__ BeamShared sh;
    pdl_wait();
    pdl_trigger();
    const int row = blockIdx.y, part = blockIdx.x, group = row / p.width;
    if (p.ended && p.ended[row]) return;
    const T* x = static_cast<const T*>(p.logits) + (size_t)group * p.group_stride + (size_t)(row - group * p.width) * p.beam_stride;
    const size_t at = (size_t)row * p.parts + part;
    beam_part(p, x, part * p.rounds * BEAM_ROUND, sh, p.share[at], p.list + at * p.count);
}

__global__ void __launch_bounds__(BEAM_THREADS) beam_join_kernel(const __grid_constant__ BeamSelect p) {
    __shared__ BeamShared sh;
    pdl_wait();
    pdl_trigger();
    const size_t row0 = (size_t)blockIdx.x * p.width;
    beam_final(
        p, blockIdx.x, sh, [&](int w, int k) { return __ldcg(p.share + (row0 + w) * p.parts + k); },
        [&](int w, int k, int i) { return __ldcg(p.list + ((row0 + w) * p.parts + k) * p.count + i); });
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

// Bytes of a state's pieces, and how many a row has.
static int state_unit(const rotor_b200_state& s) {
    const uintptr_t all = (uintptr_t)s.data | s.row_stride | (s.segments > 1 ? s.segment_stride : 0) | s.segment_bytes;
    int unit = 16;
    while (all & (unit - 1)) unit >>= 1;
    return unit;
}
static constexpr uint64_t STATE_UNITS = 0x7fffff00u;  // most pieces of a row

// Parts of `rounds` rounds for at most `most` of them.
static void beam_split(BeamSelect& p, int most) {
    const int all = (p.vocab + BEAM_ROUND - 1) / BEAM_ROUND, parts = most < all ? most : all;
    p.rounds = (all + parts - 1) / parts;
    p.parts = (all + p.rounds - 1) / p.rounds;
}

// A group's rows on the CTAs of a cluster of up to `most`, of which the device holds `active` at a time; the estimate in us (BEAM_FIXED: bars,
// lists, cluster barriers).
constexpr double BEAM_FIXED = 7.5, BEAM_ROUND_US = 0.45;
static double beam_cluster(BeamSelect& p, int most, int active) {
    beam_split(p, p.width < most ? most / p.width : 1);
    p.cluster = p.width < most ? p.width * p.parts : most;
    const int at_once = p.cluster / p.parts, rows = (p.width + at_once - 1) / at_once;
    return (double)((p.groups + active - 1) / active) * (BEAM_FIXED + rows * (p.rounds * BEAM_ROUND_US + (rows > 1 ? 2.0 : 0.0)));
}

// Clusters of `size` that the device holds at a time.
template <typename T>
static int beam_active(int size) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(BEAM_THREADS);
    cfg.dynamicSmemBytes = BEAM_DEPTH * BEAM_ROUND * sizeof(T);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = size;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, beam_cluster_kernel<T>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
    }
    return n;
}

// The form of a call: a cluster where that takes up to 13 us (the second launch and its workspace cost the host more than they save the
// GPU), else two launches with the parts that take the shortest, three CTAs on an SM and a CTA's fixed part taken as six rounds.
constexpr double BEAM_CLUSTER_US = 13.0;
static void beam_plan(BeamSelect& p, int of8, int of16) {
    BeamSelect c = p, d = p;
    double us = of8 > 0 ? beam_cluster(c, 8, of8) : 1e30;
    if (of16 > 0) {
        const double more = beam_cluster(d, BEAM_CLUSTER, of16);
        if (more < us) {
            us = more;
            c = d;
        }
    }
    if (us <= BEAM_CLUSTER_US) {
        p = c;
    } else {
        const int rows = p.groups * p.width;
        const long long slots = 3LL * fused_sm_count();
        long long best = -1;
        for (int parts = 1; parts <= 32; ++parts) {
            beam_split(c, parts);
            const long long cost = ((long long)rows * c.parts + slots - 1) / slots * (6 + c.rounds);
            if (best < 0 || cost < best) {
                best = cost;
                p.parts = c.parts;
                p.rounds = c.rounds;
            }
        }
        p.cluster = 0;
    }
    p.per_row = FastDiv(p.parts * p.count);
}

template <typename T>
static int beam_prepare(BeamSelect& p) {
    constexpr int smem = BEAM_DEPTH * BEAM_ROUND * sizeof(T);
    struct Active {
        bool known;
        int of8, of16;
    };
    static PerDevice<Active> active;
    Active& n = active.here();
    if (!n.known) {
        RB_CUDA(cudaFuncSetAttribute(beam_part_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        RB_CUDA(cudaFuncSetAttribute(beam_cluster_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        RB_CUDA(cudaFuncSetAttribute(beam_cluster_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        n.of8 = beam_active<T>(8);
        n.of16 = beam_active<T>(BEAM_CLUSTER);
        n.known = true;
    }
    beam_plan(p, n.of8, n.of16);
    return ROTOR_B200_OK;
}

static size_t beam_workspace(const BeamSelect& p) {
    return p.cluster ? 0 : (size_t)p.groups * p.width * p.parts * (sizeof(float2) + p.count * sizeof(uint2));
}

template <typename T>
static int beam_run(BeamSelect& p, void* workspace, size_t workspace_bytes, cudaStream_t st) {
    constexpr int smem = BEAM_DEPTH * BEAM_ROUND * sizeof(T);
    if (const int e = beam_prepare<T>(p)) return e;
    if (p.cluster) return launch_chained(beam_cluster_kernel<T>, dim3(p.cluster * p.groups), BEAM_THREADS, smem, st, p.cluster, p);
    if (!workspace || workspace_bytes < beam_workspace(p)) return ROTOR_B200_ERR_WORKSPACE;
    p.list = static_cast<uint2*>(workspace);
    p.share = reinterpret_cast<float2*>(p.list + (size_t)p.groups * p.width * p.parts * p.count);
    const int e = launch_chained(beam_part_kernel<T>, dim3(p.parts, p.groups * p.width), BEAM_THREADS, smem, st, 1, p);
    return e ? e : launch_chained(beam_join_kernel, dim3(p.groups), BEAM_THREADS, 0, st, 1, p);
}
static bool beam_shape(int groups, int width, int vocab, int count) {
    return groups > 0 && width > 0 && vocab > 0 && count > 0 && width <= BEAM_WIDTH && count <= BEAM_COUNT &&
           vocab <= (1 << 30) && (long long)width * vocab < (1LL << 31) && count <= (long long)width * vocab && (long long)groups * width <= 65535;
}

}  // namespace rb

using namespace rb;

extern "C" {

size_t rotor_b200_beam_select_workspace_bytes(int dtype, int groups, int width, int vocab, int count) {
    if (dtype < ROTOR_B200_F32 || dtype > ROTOR_B200_F16 || !beam_shape(groups, width, vocab, count)) return 0;
    BeamSelect p = {};
    p.groups = groups;
    p.width = width;
    p.vocab = vocab;
    p.count = count;
    const int e = dtype == ROTOR_B200_F32    ? beam_prepare<float>(p)
                  : dtype == ROTOR_B200_BF16 ? beam_prepare<__nv_bfloat16>(p)
                                             : beam_prepare<__half>(p);
    const size_t need = e ? 0 : beam_workspace(p);
    return need > 16 ? need : 16;
}

int rotor_b200_beam_select(const void* logits, int dtype, int64_t group_stride, int64_t beam_stride, const float* scores,
                           const uint8_t* ended, int groups, int width, int vocab, int count, int64_t pad, float* out_scores,
                           int64_t* out_beams, int64_t* out_tokens, void* workspace, size_t workspace_bytes, void* stream) {
    RB_REQUIRE(logits && scores && out_scores && out_beams && out_tokens && ((uintptr_t)workspace & 15) == 0);
    RB_REQUIRE(dtype >= ROTOR_B200_F32 && dtype <= ROTOR_B200_F16 && group_stride >= 0 && beam_stride >= 0);
    RB_REQUIRE(!ended || (pad >= 0 && pad < vocab));
    if (!beam_shape(groups, width, vocab, count)) return ROTOR_B200_ERR_SHAPE;
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
    p.pad = ended ? pad : 0;
    p.out_scores = out_scores;
    p.out_beams = reinterpret_cast<long long*>(out_beams);
    p.out_tokens = reinterpret_cast<long long*>(out_tokens);
    const cudaStream_t st = as_stream(stream);
    switch (dtype) {
        case ROTOR_B200_F32: return beam_run<float>(p, workspace, workspace_bytes, st);
        case ROTOR_B200_BF16: return beam_run<__nv_bfloat16>(p, workspace, workspace_bytes, st);
        default: return beam_run<__half>(p, workspace, workspace_bytes, st);
    }
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
    for (int i = 0; i < n; ++i)  // (a refused call has moved none of the states)
        if (states[i].segment_bytes / state_unit(states[i]) > STATE_UNITS / states[i].segments) return ROTOR_B200_ERR_SHAPE;
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
            const int unit = state_unit(s);
            const uint64_t per = s.segment_bytes / unit, units = per * s.segments;
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
