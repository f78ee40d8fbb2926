// Prompts over the 4-bit cache, on the fifth-generation tensor cores: causal softmax attention of many tokens a sequence over the cache's
// positions made dense (bf16 or float16 rows, cache4.cu), with windows and sinks.
//
// A CTA per SM walks the items, two blocks of 128 query rows (row = token x query head of the group) of one KV head each, those that see the
// most keys first; keys 128 at a time from the first one that an item's first token sees.  Tensor memory holds two score blocks and two
// output blocks, 512 columns in all:
//   S_w = Q_w K^T : Q_w and K tile by TMA
//   O_w += P_w V  : P_w from tensor memory (written over S_w), V tile by TMA as it lies in the dense rows
// A thread of warps 4 .. 11 owns a row of its block: it reads its 128 scores, masks them where the tile reaches over what the row sees, and
// writes 128 weights back, half of them at a time, so that the sums over the first half start while the second is made; no row is exchanged
// between threads.  While one block's scores become weights, the tensor cores work for the other, and while a block's outputs are read, its
// next queries arrive.  Outputs stay in tensor memory: the reference that weights are relative to moves, and the sums are scaled, only where a
// row's maximum has grown by more than 2^8 (weights are at most that, in float16 2^15; the sum of weights is float32).  Warp 0: TMA; warp 1: MMA issue, all of
// one thread and executed in the order of issue: the scores of a tile overwrite weights that an MMA issued before reads.  The eight warps take
// registers that the other four give back (216 and 72 of 168 each at launch; with 40 for the four the thread that issues spilled, 2% of the
// time).
// Bound: a tile of both blocks takes the tensor cores 2048 clocks and 3600 in all.  The chain of a block is weights (1900 clocks for 128 x 128:
// 550 instructions a warp, and the other block's warps share the schedulers) -> sums -> next scores (1024 clocks of MMA, some 600 of barriers:
// a barrier operation queues behind the special function unit's, 250 clocks).  Measured, bf16, 32 query and 8 KV heads of 128, causal, with the
// dense rows made first: 8192 tokens of one sequence 501 us (1.10 PFLOP/s), 8 x 2048 tokens of 20 and 5 heads 184 to 190 us (0.92); float16
// 186 to 207, most behind other work, so that the clock may be the reason (not looked into).
// Tried and slower: outputs by 16 bytes (3%: halves of sectors); weights in one piece (3%); half or a quarter of the exponentials by
// polynomials in the FMA pipe (10%, 0%); steps of 64 keys with two score blocks in flight for each block (30%: twice the barriers); items in
// the same order for every round of CTAs (8%); weights against the last reference with a look at their sum afterwards, without the tile's
// maximum (4 to 9%).
// Rounded to the 16-bit type, beside the outputs: keys and values as dense rows (the tensor cores' operands) and weights (their sum is
// of unrounded ones); scores, maxima, sums and outputs are float32.
// Waits are bounded; a wait that runs out records a code in the library status word, the CTA stops issuing work, frees its tensor memory
// and returns.  No multicast, this GPU's memory only.
#include <cstdlib>

#include "cache4.cuh"
#include "tc5.cuh"

namespace rb {

constexpr int P4_ROWS = 128, P4_KEYS = 128, P4_THREADS = 384;
constexpr int P4_SOFT_REGS = 216, P4_OTHER_REGS = 72, P4_REGS = 168;  // 2 x 128 x 216 + 128 x 72 = 384 x 168
// The reference of a row's weights: its maximum less LIFT powers of two, kept while the maximum is below it plus LIFT and SLACK.  bf16 weights have
// float32's range; float16 ones end at 2^15 with this, and the smallest are 2^-32 of the largest instead of 2^-25 (131072 positions at 2^-25.5
// beside one of 2^0 are 0.3 % of the mass).
constexpr float P4_SLACK = 8.f;
template <bool HALF>
constexpr float P4_LIFT = HALF ? 7.f : 0.f;

template <int DK>
struct P4Cfg {
    // two query blocks, and a ring of tiles that keys and values take in turn: of 128 columns as many as fit
    static constexpr int TILE = P4_KEYS * DK * 2, SLOTS = DK == 128 ? 5 : 8, SMEM = (2 + SLOTS) * TILE + 1024;
};

struct P4Params {
    uint16_t* out;
    const int* past_len;
    const float* sinks;
    unsigned* status;
    int heads, kv_heads, dim, seq, span, max_seq, window;
    int blocks, items;              // of 2 x 128 rows: of a sequence's KV head, of the call
    bool whole;                     // outputs begin at a multiple of 32 bytes
    float scale2;                   // |scale| log2(e) (its sign is in the keys)
};

__device__ __forceinline__ void p4_tma_q(uint32_t dst, const CUtensorMap* map, int x, int head, int token, int b, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(head), "r"(token), "r"(b), "r"(bar)
        : "memory");
}

template <bool HALF>
__device__ __forceinline__ uint32_t p4_pack(float a, float b) {
    return HALF ? pack_half(a, b) : t5_pack(a, b);
}

// Item i of a call: the blocks of late tokens, which see more keys, come first.  CTAs take a round of items in one order and the next round
// in the other, so that none gets the longest of every round.
__device__ __forceinline__ int p4_item(int round) {
    const int first = round * (int)gridDim.x;
    return round & 1 ? first + (int)gridDim.x - 1 - (int)blockIdx.x : first + (int)blockIdx.x;
}

struct P4Item {
    int b, hk, s0, s_last, past, kb0, ntiles;
    __device__ __forceinline__ P4Item(const P4Params& p, int i) {
        const int QT = P4_ROWS / (p.heads / p.kv_heads), per = p.items / p.blocks;  // tokens of a block; (sequence, KV head) pairs
        const int block = p.blocks - 1 - i / per, pair = i % per;
        b = pair / p.kv_heads;
        hk = pair - b * p.kv_heads;
        s0 = block * 2 * QT;
        s_last = min(s0 + 2 * QT, p.seq) - 1;
        past = __ldcg(p.past_len + b);
        kb0 = first_visible(past + s0, 0, p.window);
        const int t_end = min(past + s_last + 1, p.max_seq);
        ntiles = t_end > kb0 ? (t_end - kb0 + P4_KEYS - 1) / P4_KEYS : 0;
    }
};

template <int DK, bool HALF>
__global__ void __launch_bounds__(P4_THREADS, 1)
cache4_prompt_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ P4Params p) {
    using C = P4Cfg<DK>;
    extern __shared__ unsigned char p4_raw[];
    __shared__ __align__(8) unsigned long long s_full[C::SLOTS], s_empty[C::SLOTS], s_sfull[2], s_pfull[2][2], s_done[2], s_qfull[2], s_qempty[2];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    const uint32_t qbase = (smem_u32(p4_raw) + 1023u) & ~1023u, ring = qbase + 2 * C::TILE;
    // keys of the CTA's tile t are load 2 t, values load 2 t + 1
    auto slot_of = [](uint32_t load) { return load % C::SLOTS; };
    auto parity_of = [](uint32_t load) { return load / C::SLOTS & 1u; };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = p.heads / p.kv_heads, QT = P4_ROWS / G;  // tokens of a block
    volatile int* abort_flag = &s_abort;

    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < C::SLOTS; ++s) {
            t5_bar_init(smem_u32(&s_full[s]), 1);
            t5_bar_init(smem_u32(&s_empty[s]), 1);
        }
        for (int s = 0; s < 2; ++s) {
            t5_bar_init(smem_u32(&s_sfull[s]), 1);
            t5_bar_init(smem_u32(&s_pfull[s][0]), 4);
            t5_bar_init(smem_u32(&s_pfull[s][1]), 4);
            t5_bar_init(smem_u32(&s_done[s]), 1);
            t5_bar_init(smem_u32(&s_qfull[s]), 1);
            t5_bar_init(smem_u32(&s_qempty[s]), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;  // S_0 [0, 128)  S_1 [128, 256)  O_0 [256, 256 + DK)  O_1 [384, 384 + DK)

    if (warp >= 4) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(P4_SOFT_REGS));
        const int w = (warp >> 2) - 1, r = (warp & 3) * 32 + lane;  // block and row
        const int in_block = r / G, gi = r - in_block * G;
        const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t sbuf = lane_base + (uint32_t)w * 128u, obuf = lane_base + 256u + (uint32_t)w * 128u;
        const float2 scale = make_float2(p.scale2, p.scale2);
        bool ok = true;
        uint32_t tile = 0;  // of the CTA, over its items
        for (int round = 0; ok && p4_item(round) < p.items; ++round) {
            const P4Item it(p, p4_item(round));
            const int token = it.s0 + w * QT + in_block, pos = it.past + min(token, it.s_last);
            const bool real = in_block < QT && token <= it.s_last;
            const int lo = first_visible(pos, 0, p.window), hi = min(pos, p.max_seq - 1);  // visible keys [lo, hi]
            float ref = -INFINITY, mass = 0.f;
            for (int j = 0; j < it.ntiles; ++j, ++tile) {
                ok = __all_sync(0xffffffffu, t5_wait(smem_u32(&s_sfull[w]), tile & 1u, abort_flag, p.status, 0x7b000001u));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t s[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) t5_ld32(sbuf + 32u * c, s[c]);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                const int kb = it.kb0 + j * P4_KEYS;
                if (kb < lo || kb + P4_KEYS - 1 > hi) {
#pragma unroll
                    for (int i = 0; i < 128; ++i)
                        if (kb + i < lo || kb + i > hi) s[i >> 5][i & 31] = 0xff800000u;
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 32; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) top[c] = fmaxf(top[c], __uint_as_float(s[c][i]));
                float m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                m = m == -INFINITY ? m : m * p.scale2;
                const bool grown = m > ref + (P4_SLACK + P4_LIFT<HALF>);
                if (__any_sync(0xffffffffu, grown)) {
                    const float now = grown ? m - P4_LIFT<HALF> : ref, alpha = grown ? fast_exp2(ref - now) : 1.f;
                    ref = now;
                    mass *= alpha;
                    if (j > 0) {  // (the first tile's sums begin at zero)
                        ok = __all_sync(0xffffffffu, t5_wait(smem_u32(&s_done[w]), (tile - 1u) & 1u, abort_flag, p.status, 0x7b000002u));
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                        for (int c = 0; c < DK; c += 32) {
                            uint32_t o[32];
                            t5_ld32(obuf + c, o);
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            t5_st32(obuf + c, o);
                        }
                    }
                }
                const float base = ref == -INFINITY ? 0.f : -ref;  // (no key of this row yet)
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t pk[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int k = h * 64 + 2 * i;
                        const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[k >> 5][k & 31]), __uint_as_float(s[k >> 5][(k & 31) + 1])), scale,
                                                    make_float2(base, base));
                        const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
                        sum[i & 1] = __fadd2_rn(sum[i & 1], e);
                        pk[i] = p4_pack<HALF>(e.x, e.y);
                    }
                    t5_st32(sbuf + (uint32_t)h * 32u, pk);  // 128 weights in columns [0, 64) of the scores' block
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) t5_bar_arrive(smem_u32(&s_pfull[w][h]));
                }
                mass += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            }
            if (ok && it.ntiles > 0)
                ok = __all_sync(0xffffffffu, t5_wait(smem_u32(&s_done[w]), (tile - 1u) & 1u, abort_flag, p.status, 0x7b000003u));
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float inv = ref == -INFINITY && mass == mass ? 0.f : 1.f / mass;  // (no key: zeros)
            if (p.sinks && real) {
                const float sink = __ldg(p.sinks + it.hk * G + gi) * 1.4426950408889634f, most = fmaxf(ref, sink), mine = fast_exp2(ref - most);
                inv = ref == -INFINITY && mass == mass ? 0.f : mine / (mass * mine + fast_exp2(sink - most));
            }
            uint16_t* out = p.out + (((size_t)it.b * p.seq + (real ? token : 0)) * p.heads + it.hk * G + gi) * p.dim;
#pragma unroll
            for (int c = 0; c < DK; c += 32) {
                uint32_t o[32];
                if (it.ntiles > 0) {
                    t5_ld32(obuf + c, o);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0u;
                }
                if (real && c < p.dim) {
#pragma unroll
                    for (int i = 0; i < 32; i += 16) {
                        uint32_t v[8];
#pragma unroll
                        for (int n = 0; n < 8; ++n) {
                            const float a = __uint_as_float(o[i + 2 * n]) * inv, c = __uint_as_float(o[i + 2 * n + 1]) * inv;
                            v[n] = HALF ? pack_half_finite(a, c) : t5_pack(a, c);
                        }
                        if (p.whole) {
                            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + c + i), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                                         "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                                         : "memory");
                        } else {
                            *reinterpret_cast<uint4*>(out + c + i) = make_uint4(v[0], v[1], v[2], v[3]);
                            *reinterpret_cast<uint4*>(out + c + i + 8) = make_uint4(v[4], v[5], v[6], v[7]);
                        }
                    }
                }
            }
            // (the next item's first P V overwrites these columns after this block's next weights have been announced)
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(P4_OTHER_REGS));
        if (warp == 0 && elect_lane()) {
            uint32_t load = 0, nth = 0;  // of the CTA
            bool ok = true;
            for (int round = 0; ok && p4_item(round) < p.items; ++round) {
                const P4Item it(p, p4_item(round));
                if (it.ntiles == 0) continue;
                const int row0 = (it.b * p.kv_heads + it.hk) * p.span + it.kb0;
                auto queries = [&](int w) {
                    if (!t5_wait(smem_u32(&s_qempty[w]), (nth & 1u) ^ 1u, abort_flag, p.status, 0x7b000004u)) return false;
                    const uint32_t bar = smem_u32(&s_qfull[w]);
                    t5_bar_expect(bar, QT * G * DK * 2);
#pragma unroll
                    for (int pn = 0; pn < DK / 64; ++pn)
                        p4_tma_q(qbase + w * C::TILE + pn * 16384, &tm_q, pn * 64, it.hk * G, it.s0 + w * QT, it.b, bar);
                    return true;
                };
                ok = queries(0) && queries(1);
                ++nth;
                for (int j = 0; j < 2 * it.ntiles && ok; ++j, ++load) {  // keys and values of a tile, in turn
                    const uint32_t slot = slot_of(load), bar = smem_u32(&s_full[slot]);
                    ok = t5_wait(smem_u32(&s_empty[slot]), parity_of(load) ^ 1u, abort_flag, p.status, 0x7b000005u);
                    if (!ok) break;
                    t5_bar_expect(bar, C::TILE);
#pragma unroll
                    for (int pn = 0; pn < DK / 64; ++pn)
                        t5_tma_2d(ring + slot * C::TILE + pn * 16384, j & 1 ? &tm_v : &tm_k, pn * 64, row0 + (j >> 1) * P4_KEYS, bar);
                }
            }
        } else if (warp == 1 && elect_lane()) {
            constexpr uint32_t idesc_s = HALF ? t5_idesc_f16(128, P4_KEYS) : t5_idesc_bf16(128, P4_KEYS);
            constexpr uint32_t idesc_o = HALF ? t5_idesc_f16(128, DK, true) : t5_idesc_bf16(128, DK, true);
            // scores of block w and the CTA's tile t; `last`: of the item, whose queries are read for the last time
            auto issue_s = [&](int w, uint32_t t, bool last) {
                const uint64_t dq = t5_desc(qbase + w * C::TILE), dk = t5_desc(ring + slot_of(2 * t) * C::TILE);
#pragma unroll
                for (int k16 = 0; k16 < DK / 16; ++k16) {
                    const uint64_t off = (uint64_t)(((k16 >> 2) * 16384 + (k16 & 3) * 32) >> 4);
                    t5_mma_ss(tmem + (uint32_t)w * 128u, dq + off, dk + off, idesc_s, k16 > 0);
                }
                t5_commit(smem_u32(&s_sfull[w]));
                if (w == 1) t5_commit(smem_u32(&s_empty[slot_of(2 * t)]));
                if (last) t5_commit(smem_u32(&s_qempty[w]));
            };
            auto issue_pv = [&](int w, uint32_t t, int half, bool first) {
                const uint64_t dv = t5_desc_mn(ring + slot_of(2 * t + 1) * C::TILE, 16384);
#pragma unroll
                for (int k = 0; k < P4_KEYS / 32; ++k) {
                    const int k16 = half * (P4_KEYS / 32) + k;
                    t5_mma_ts(tmem + 256u + (uint32_t)w * 128u, tmem + (uint32_t)w * 128u + (uint32_t)k16 * 8u, dv + (uint64_t)(k16 * 2048 >> 4), idesc_o,
                              !first || k16 > 0);
                }
                if (half == 0) return;
                t5_commit(smem_u32(&s_done[w]));
                if (w == 1) t5_commit(smem_u32(&s_empty[slot_of(2 * t + 1)]));
            };
            // The tiles of the CTA's items in a row: scores of tile t + 1 are issued behind the sums of tile t, across items too.
            int round = 0, left = 0;  // left: tiles of the item after the next one to score
            uint32_t nth = 0;                 // items begun
            auto begin = [&]() {              // the next item that has tiles
                while (p4_item(round) < p.items) {
                    left = P4Item(p, p4_item(round++)).ntiles;
                    if (left > 0) {
                        ++nth;
                        return true;
                    }
                }
                return false;
            };
            bool ok = true, more = begin();
            bool first_s = true;              // the tile to score is its item's first
            auto score = [&](int w, uint32_t t) {
                if (first_s && !t5_wait(smem_u32(&s_qfull[w]), (nth - 1u) & 1u, abort_flag, p.status, 0x7b000007u)) return false;
                issue_s(w, t, left == 1);
                return true;
            };
            uint32_t t = 0;
            auto loaded = [&](uint32_t load) {
                return t5_wait(smem_u32(&s_full[slot_of(load)]), parity_of(load), abort_flag, p.status, 0x7b000008u);
            };
            if (more) ok = loaded(0) && score(0, 0) && score(1, 0);
            bool first_pv = true;             // the tile to sum is its item's first
            while (more && ok) {
                const bool ends = left == 1;  // tile t is its item's last
                if (!ends) {
                    --left;
                    first_s = false;
                } else {
                    more = begin();
                    first_s = true;
                }
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    if (ok && w == 0) ok = loaded(2 * t + 1) && (!more || loaded(2 * t + 2));
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if (ok) ok = t5_wait(smem_u32(&s_pfull[w][half]), t & 1u, abort_flag, p.status, 0x7b000009u);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        issue_pv(w, t, half, first_pv);
                    }
                    if (!ok) break;
                    if (more) ok = score(w, t + 1);
                }
                first_pv = ends;
                ++t;
            }
        }
    }

    // ---------------- common exit: nothing of this CTA may still be in flight when it returns
    if (*abort_flag && threadIdx.x == 0) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) {
        }  // about a millisecond for copies already issued to land
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 0) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

bool prompt_attn_supported(int batch, int heads, int kv_heads, int dim, int span) {
    static const bool off = getenv("ROTOR_B200_NO_TCGEN05") != nullptr;
    return !off && dim <= 128 && heads / kv_heads <= P4_ROWS && batch <= 65535 && kv_heads <= 65535 && (size_t)batch * kv_heads * span <= 0x7fffffffu;
}

// Queries [batch][seq][heads][dim] of any strides; a box is a block's tokens and the group's heads, 64 columns.
static bool p4_map_q(CUtensorMap* map, const PromptAttn& p, int G, int QT) {
    T5EncodeFn enc = t5_encoder();
    const cuuint64_t gdim[4] = {(cuuint64_t)p.dim, (cuuint64_t)p.heads, (cuuint64_t)p.seq, (cuuint64_t)p.batch};
    const size_t strides[3] = {p.heads > 1 ? p.q_head : (size_t)p.dim, p.seq > 1 ? p.q_row : (size_t)p.heads * p.dim,
                               p.batch > 1 ? p.q_seq : (size_t)p.heads * p.dim * p.seq};
    const cuuint64_t gstride[3] = {(cuuint64_t)strides[0] * 2, (cuuint64_t)strides[1] * 2, (cuuint64_t)strides[2] * 2};
    const cuuint32_t box[4] = {64u, (cuuint32_t)G, (cuuint32_t)QT, 1u}, estride[4] = {1u, 1u, 1u, 1u};
    return enc && enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(p.q), gdim, gstride, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DK, bool HALF>
static int p4_go(const PromptAttn& p, const P4Params& a, cudaStream_t st) {
    static PerDevice<bool> once;
    if (!once.here()) {
        // the kernel's warps share out the registers they were launched with: without all of them they would wait for ever
        cudaFuncAttributes f;
        RB_CUDA(cudaFuncGetAttributes(&f, cache4_prompt_kernel<DK, HALF>));
        if (f.numRegs < P4_REGS) return ROTOR_B200_ERR_CUDA;
        RB_CUDA(cudaFuncSetAttribute(cache4_prompt_kernel<DK, HALF>, cudaFuncAttributeMaxDynamicSharedMemorySize, P4Cfg<DK>::SMEM));
        once.here() = true;
    }
    const size_t rows = (size_t)p.batch * p.kv_heads * p.span;
    const int G = p.heads / p.kv_heads;
    CUtensorMap tq, tk, tv;
    if (!p4_map_q(&tq, p, G, P4_ROWS / G) || !t5_map_bf16(&tk, p.k, rows, p.dim, p.dim, P4_KEYS) || !t5_map_bf16(&tv, p.v, rows, p.dim, p.dim, P4_KEYS))
        return ROTOR_B200_ERR_CUDA;
    const int grid = a.items < fused_sm_count() ? a.items : fused_sm_count();
    cache4_prompt_kernel<DK, HALF><<<grid, P4_THREADS, P4Cfg<DK>::SMEM, st>>>(tq, tk, tv, a);
    return launch_status();
}

int launch_prompt_attn(const PromptAttn& p, cudaStream_t st) {
    if (!prompt_attn_supported(p.batch, p.heads, p.kv_heads, p.dim, p.span)) return ROTOR_B200_ERR_SHAPE;
    P4Params a = {};
    a.out = static_cast<uint16_t*>(p.out);
    a.whole = ((uintptr_t)p.out & 31) == 0;
    a.past_len = p.past_len;
    a.sinks = p.sinks;
    a.status = library_status_word();
    if (!a.status) return ROTOR_B200_ERR_CUDA;
    a.heads = p.heads;
    a.kv_heads = p.kv_heads;
    a.dim = p.dim;
    a.seq = p.seq;
    a.span = p.span;
    a.max_seq = p.max_seq;
    a.window = p.window;
    const int tokens = 2 * (P4_ROWS / (p.heads / p.kv_heads));
    a.blocks = (p.seq + tokens - 1) / tokens;
    const long long items = (long long)a.blocks * p.kv_heads * p.batch;
    if (items > 0x3fffffff) return ROTOR_B200_ERR_SHAPE;
    a.items = (int)items;
    a.scale2 = fmaxf(fabsf(p.scale) * 1.4426950408889634f, 1e-30f);  // (a masked score, -inf, times zero would be no number)
    if (p.half) return p.dim <= 64 ? p4_go<64, true>(p, a, st) : p4_go<128, true>(p, a, st);
    return p.dim <= 64 ? p4_go<64, false>(p, a, st) : p4_go<128, false>(p, a, st);
}

}  // namespace rb
