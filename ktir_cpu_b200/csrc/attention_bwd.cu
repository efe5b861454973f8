// Gradients of attention: with S = scale Q K^T, P = exp(S - lse) where a query sees a key, D = rowsum(dO * O),
//   dS = P * (dO V^T - D),   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO.
// It takes over the loops of a KTIR program that walks tiles of keys for dQ and tiles of queries for dK and dV
// (linalg.matmul, exp, select and linalg.reduce per pair of tiles; ktir_cpu/ops/arith_ops.py:323-340,
// ktir_cpu/dialects/linalg_ops.py:136-347).
//
// The tensor cores bound it: five products of 2 * 128 * 128 * head_dim operations per pair of 128-row tiles are needed.
// Seven are made here: a CTA owns a tile of keys (S^T, dO V^T transposed, dV, dK) or one of queries (S, dO V^T, dQ), so that
// every sum has one owner and one order, and no partial sum of dQ crosses HBM.  The kernel is persistent, and a CTA that is done
// takes the next tile, longest walks first.
//
// Both kinds of tile are the same loop.  A CTA holds two tiles of 128 rows X and Y (K and V, or Q and dO) in shared memory and
// streams pairs of 64-row tiles X', Y' (Q and dO, or K and V) through a ring by TMA.  Per step one warp issues
// S = X X'^T and T = Y Y'^T into a slot of TMEM (there are two at 128 columns a head, three at 64); a warpgroup reads them, a thread
// a row (two take the steps in turn), and writes P and dS as f16 over the same columns; the next products take them from there
// as their A operand: acc0 += dS X' and, for keys, acc1 += P Y'.  While one step is in the softmax, the tensor core has the
// other slots'.
//
// f16 operands.  P is at most 1 but mostly near 1 / keys, dS is as small as the gradient: both are rounded to f16 (2^-12 of the
// value on average; exp2 is approximate to 2^-22, all else before the results is f32) after a shift by powers of two that keeps
// them in range: P by 2^14, dS by 2^14 / B with B >= |dO V^T - D| a power of two from the norms of dO and V: for dQ, whose sums
// run over keys, per query and from the keys that it sees, for dK per key and from the queries that see it.  (From all of a head,
// dK of the keys behind a query 10^6 times as loud as the others lost 2 % of its value, dQ of the queries before such a value
// likewise.)  Sums, D and the statistics are f32.  Where few rows see a key these roundings are multiplied too (MODE 2).
//
// 256 heads of 2048 positions, 128 wide, causal: 1.03 ms, 667 TFLOP/s of the five products (933 of the seven), 1.20 ms once
// the power cap holds; 16 / 4 heads of 8192 positions 0.76 ms, 906, capped 0.88.
#include <type_traits>

#include "tc_common.cuh"

#define AB_M 128                   // rows that a CTA owns
#define AB_N 64                    // streamed rows of a step
#define AB_SHIFT 14.f
#define AB_LOG2E 1.4426950408889634f

// A kernel that follows another on its stream may start while that one ends, up to where it waits; `ab_follow` allows it.
static __device__ __forceinline__ void ab_follow() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
static __device__ __forceinline__ void ab_wait_for_rows() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- what the rows bring: 14 - lse / ln 2, D and |dO| per query, |V| per key, and the largest norms of a block of rows --
// HBM bounds it (O, dO and V once; 256 heads of 2048 positions, 128 wide: 81 us, 5.0 TB/s).  A block takes
// BLOCK rows of heads, 2^heads_log neighbouring heads of BLOCK >> heads_log positions (so that what it reads lies together),
// head_dim / 8 threads each, four of their loads ahead of the arithmetic.
struct ab_scratch {
    unsigned* taken;               // items handed out beyond the first of every CTA
    float* neg_lse;                // [heads][padded queries]
    float* d;
    float* norm;
    float2* most_q;                // [heads][q_blocks]: largest |dO| and |D| of a block of queries
    float* most_v;                 // [key heads][k_blocks]: largest |V| of a block of keys
    float* norm_v;                 // [key heads][keys]: |V|
    int64_t padded;
    int q_log, k_log;              // heads_log for queries, for keys
    int q_blocks, k_blocks;
    int block;
};

// Dot product of eight f16 in f32.  (The fma takes f16 factors; converted first, 2048 positions of 256 heads took 92 us, not 86.)
static __device__ __forceinline__ float ab_dot8(uint4 a, uint4 b) {
    const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        asm("{\n .reg .b16 p, q, u, v;\n mov.b32 {p, q}, %1;\n mov.b32 {u, v}, %2;\n fma.rn.f32.f16 %0, p, u, %0;\n fma.rn.f32.f16 %0, q, v, %0;\n}"
            : "+f"(s) : "r"(x[i]), "r"(y[i]));
    return s;
}

template <int HD, int BLOCK>
__global__ void __launch_bounds__(256) ktb_attention_rows_kernel(const ktb_attn_bwd_args a, const ab_scratch w) {
    constexpr int LANES = HD / 8, GROUPS = 256 / LANES, BATCH = 4;
    ab_follow();
    if (blockIdx.x == 0 && threadIdx.x == 0) *w.taken = 0;
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const __half* base = reinterpret_cast<const __half*>(a.arena);
    const int kv_heads = a.heads / a.kv_group;
    const int q_wide = (a.heads + (1 << w.q_log) - 1) >> w.q_log, k_wide = (kv_heads + (1 << w.k_log) - 1) >> w.k_log;
    const bool keys = blockIdx.x >= (unsigned)q_wide * w.q_blocks;
    const int at = keys ? blockIdx.x - q_wide * w.q_blocks : blockIdx.x, wide = keys ? k_wide : q_wide, log = keys ? w.k_log : w.q_log;
    const int block = at / wide, head0 = (at % wide) << log, heads = keys ? kv_heads : a.heads;
    const int64_t row0 = (int64_t)block * (BLOCK >> log), rows = keys ? a.kv_len : a.q_len;
    const __half* from = base + (keys ? a.v_off : a.do_off) + lane * 8;
    const __half* from_o = base + a.o_off + lane * 8;
    const int64_t stride = keys ? a.v_row : a.do_row, head_stride = keys ? a.v_head : a.do_head;
    // (a group's heads are all the same one when there are no more heads side by side than groups)
    const int head = head0 + (group & ((1 << log) - 1));
    float most = 0.f, most_d = 0.f;
#pragma unroll 1
    for (int i0 = 0; i0 < BLOCK; i0 += BATCH * GROUPS) {
        uint4 g[BATCH], o[BATCH];
        float lse[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int64_t row = row0 + ((i0 + i * GROUPS + group) >> log);
            g[i] = o[i] = make_uint4(0, 0, 0, 0);
            lse[i] = -INFINITY;
            if (row < rows && head < heads && i0 + i * GROUPS + group < BLOCK) {
                g[i] = *reinterpret_cast<const uint4*>(from + row * stride + head * head_stride);
                if (!keys) {
                    o[i] = *reinterpret_cast<const uint4*>(from_o + row * a.o_row + head * a.o_head);
                    lse[i] = (reinterpret_cast<const float*>(a.arena) + a.lse_off)[row * a.lse_row + (int64_t)head * a.lse_head];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int64_t row = row0 + ((i0 + i * GROUPS + group) >> log);
            float g2 = ab_dot8(g[i], g[i]), d = ab_dot8(g[i], o[i]);
#pragma unroll
            for (int x = LANES / 2; x; x >>= 1) {
                g2 += __shfl_xor_sync(0xffffffffu, g2, x);
                d += __shfl_xor_sync(0xffffffffu, d, x);
            }
            g2 = g2 <= 3.0e38f ? g2 : 0.f;                              // (a row with an infinity has no say in the shift)
            most = fmaxf(most, g2);
            if (fabsf(d) <= 3.0e38f) most_d = fmaxf(most_d, fabsf(d));
            if (!keys && lane == 0 && row < w.padded && head < heads && i0 + i * GROUPS + group < BLOCK) {
                const int64_t to = (int64_t)head * w.padded + row;
                // (no probability: rows past the end, rows that see nothing)
                w.neg_lse[to] = lse[i] == -INFINITY ? -INFINITY : fmaf(-lse[i], AB_LOG2E, AB_SHIFT);
                w.d[to] = d;
                w.norm[to] = sqrtf(g2);
            }
            if (keys && lane == 0 && row < rows && head < heads && i0 + i * GROUPS + group < BLOCK) w.norm_v[head * rows + row] = sqrtf(g2);
        }
    }
    __shared__ float sa[GROUPS], sd[GROUPS];
    if (lane == 0) {
        sa[group] = most;
        sd[group] = most_d;
    }
    __syncthreads();
    const int mine = threadIdx.x;
    if (mine < (1 << log) && head0 + mine < heads) {
        most = most_d = 0.f;
        for (int i = mine; i < GROUPS; i += 1 << log) {
            most = fmaxf(most, sa[i]);
            most_d = fmaxf(most_d, sd[i]);
        }
        if (keys) w.most_v[(int64_t)(head0 + mine) * w.k_blocks + block] = sqrtf(most);
        else w.most_q[(int64_t)(head0 + mine) * w.q_blocks + block] = make_float2(sqrtf(most), most_d);
    }
}

// A power of two s with |x| s <= 1 for |x| <= bound.
static __device__ __forceinline__ float ab_shrink(float bound) {
    const int e = (int)((__float_as_uint(bound) >> 23) & 255) - 127;            // bound < 2^(e + 1)
    if (!(bound > 0.f) || e < -120) return bound > 0.f ? 0x1p100f : 1.f;
    return __uint_as_float((unsigned)(127 - (e + 1)) << 23);
}

// ---- the kernel ----------------------------------------------------------------------------------------------------
template <int HD>
struct ab_shape {
    static constexpr int BLOCKS = HD / 64;                  // 64-column blocks of a tile (a 128-byte swizzled row each)
    static constexpr int OWN = AB_M * HD * 2;               // bytes of X, of Y
    static constexpr int STEP = AB_N * HD * 2;              // bytes of X', of Y'
    static constexpr int STAGES = HD == 64 ? 8 : 4;         // 128 KB of the stream on its way
    static constexpr size_t SMEM = 2 * OWN + STAGES * (2 * STEP + 3 * AB_N * 4) + 8 * 2048 + 1024 + 512;
    // columns of TMEM: two accumulators (for queries X and Y as f16 pairs in place of the second), then the slots: S and T
    static constexpr int ACC1 = HD, X = HD, Y = HD + HD / 2, SLOT = 2 * HD;
    static constexpr int SLOTS = (512 - SLOT) / (2 * AB_N);
    // With two slots a step's way from its scores to its sums and back is what a step takes: it is cut in two (see the softmax).
    // Where three slots hide it the cut only costs barriers (64 wide, a step of keys 0.60 us, cut 0.62; 128 wide 0.88, cut 0.79).
    static constexpr bool CUT = SLOTS < 3;
};

// Waits for a phase no matter what else has failed, so that no copy is under way into memory that the CTA gives up.
static __device__ void ab_drain(uint64_t* bar, uint32_t parity) {
    const long long start = clock64();
    while (!tc_mbar_try_wait(bar, parity))
        if (clock64() - start > 1000000000ll) return;
}

// What there is to do: the tiles of keys, then those of queries; among each, longest walks first, either head by head (so that
// the CTAs at work share their streams in L2) or over all heads (where there are few tiles and a long one must not come last).
// A walk may be cut into parts, where a few long ones would leave most SMs idle; the parts' sums are joined afterwards.
struct ab_work {
    int key_tiles, key_heads, key_parts, query_tiles, query_heads, query_parts;
    int by_head;
    int twice;                                              // every step comes twice (only where PARTS)
    float *part_k, *part_v, *part_q;                        // [part][row][head][head_dim] of the rows and heads that are wanted
    template <bool PARTS> __device__ __forceinline__ int of_keys() const { return key_tiles * key_heads * (PARTS ? key_parts : 1); }
    template <bool PARTS> __device__ __forceinline__ int total() const { return of_keys<PARTS>() + query_tiles * query_heads * (PARTS ? query_parts : 1); }
};

struct ab_item {
    bool keys;
    int row0, head, part;
    int first, per_head;                                    // a whole walk: per_head streamed tiles from `first` on, for every streamed head
    int skip, n;                                            // this part of it: n steps after `skip`
};

template <bool PARTS>
static __device__ __forceinline__ ab_item ab_decode(const ktb_attn_bwd_args& a, const ab_work& j, int index) {
    ab_item t;
    const int of_keys = j.of_keys<PARTS>();
    t.keys = index < of_keys;
    const int parts = t.keys ? j.key_parts : j.query_parts, tiles = t.keys ? j.key_tiles : j.query_tiles, heads = t.keys ? j.key_heads : j.query_heads;
    int at = t.keys ? index : index - of_keys;
    t.part = 0;
    if (PARTS) {
        const int whole = at / parts;
        t.part = at - whole * parts;
        at = whole;
    }
    const int rank = j.by_head ? at % tiles : at / heads, head_here = j.by_head ? at / tiles : at % heads;
    t.first = 0;
    if (t.keys) {
        t.row0 = a.dk_row0 + rank * AB_M;
        t.head = a.dk_head0 + head_here;
        t.per_head = (a.q_len + AB_N - 1) / AB_N;
        if (a.causal) {
            const long long q = (long long)t.row0 - a.causal_delta;             // the first query that sees key row0
            t.first = q <= 0 ? 0 : q >= a.q_len ? t.per_head : (int)(q / AB_N);
        }
        t.per_head -= t.first;
    } else {
        t.row0 = a.dq_row0 + (tiles - 1 - rank) * AB_M;
        t.head = a.dq_head0 + head_here;
        t.per_head = (a.kv_len + AB_N - 1) / AB_N;
        if (a.causal) {
            const int last_row = t.row0 + AB_M - 1 < a.q_len - 1 ? t.row0 + AB_M - 1 : a.q_len - 1;
            const long long key = (long long)last_row + a.causal_delta;         // the last key that the tile sees
            const long long n = key < 0 ? 0 : key / AB_N + 1;
            if (n < t.per_head) t.per_head = (int)n;
        }
    }
    t.skip = 0;
    t.n = t.per_head * (t.keys ? a.kv_group : 1);
    if (PARTS) {
        const long long steps = t.n;
        t.skip = (int)(steps * t.part / parts);
        t.n = ((int)(steps * (t.part + 1) / parts) - t.skip) << j.twice;
    }
    return t;
}

// Two values as f16, or what that rounding leaves out of them (nothing of an infinity).
template <bool RESTS>
static __device__ __forceinline__ __half2 ab_pack(float x, float y, bool rest) {
    __half2 h = __floats2half2_rn(x, y);
    if (RESTS && rest) {
        const float u = __low2float(h), v = __high2float(h);
        h = __floats2half2_rn(fabsf(u) <= 65504.f ? x - u : 0.f, fabsf(v) <= 65504.f ? y - v : 0.f);
    }
    return h;
}

// MODE: 0 whole walks, 1 parts of walks, 2 parts of walks whose steps come twice: P and dS as f16, then what that left out of them.
template <int HD, int MODE>
__global__ void __launch_bounds__(384, 1)
ktb_attention_bwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_g,
                         const ktb_attn_bwd_args a, const ab_scratch w, const ab_work work, ktb_status* st) {
    typedef ab_shape<HD> Z;
    constexpr bool PARTS = MODE > 0, TWICE = MODE == 2;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* sX = smem;
    uint8_t* sY = sX + Z::OWN;
    uint8_t* ring = sY + Z::OWN;                            // per stage X', then Y'
    float* sRow = reinterpret_cast<float*>(ring + Z::STAGES * 2 * Z::STEP);     // keys: per stage 64 x (14 - lse / ln 2), 64 x D, 64 x |dO| where steps come twice
    uint8_t* sOut = reinterpret_cast<uint8_t*>(sRow + Z::STAGES * 3 * AB_N);    // 2 KB a warp of the softmax
    uint64_t* full = reinterpret_cast<uint64_t*>(sOut + 8 * 2048);
    uint64_t *empty = full + Z::STAGES, *own_full = empty + Z::STAGES, *own_free = own_full + 1, *a_ready = own_free + 1;
    uint64_t *acc_free = a_ready + 1, *done = acc_free + 1, *next_full = done + 1, *next_free = next_full + 2;
    uint64_t *s_full = next_free + 2, *t_full = s_full + Z::SLOTS, *p_full = t_full + Z::SLOTS;     // p_full: per slot and half of its columns
    volatile int* next = reinterpret_cast<volatile int*>(p_full + 2 * Z::SLOTS);        // items handed out, two at a time
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(const_cast<int*>(next) + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int grp = a.kv_group, total = work.total<PARTS>();

    if (threadIdx.x == 0) {
        for (int i = 0; i < Z::STAGES; ++i) {
            tc_mbar_init(&full[i], 1);
            tc_mbar_init(&empty[i], 1);
        }
        tc_mbar_init(own_full, 1);
        tc_mbar_init(own_free, 1);
        tc_mbar_init(a_ready, 8);
        tc_mbar_init(acc_free, 8);
        tc_mbar_init(done, 1);
        for (int i = 0; i < 2; ++i) {
            tc_mbar_init(&next_full[i], 1);
            tc_mbar_init(&next_free[i], 10);                // warps 1 and 2, eight warps of the softmax
        }
        for (int i = 0; i < Z::SLOTS; ++i) {
            tc_mbar_init(&s_full[i], 1);
            tc_mbar_init(&t_full[i], 1);
            tc_mbar_init(&p_full[2 * i], 4);
            tc_mbar_init(&p_full[2 * i + 1], 4);
        }
        *abort_flag = 0;
        tc_fence_barrier_init();
    }
    __syncthreads();
    if (warp == 1) tc_tmem_alloc(tmem_slot, 512);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

    // The k-th item of this CTA (whichever CTA is free takes the next one; what is computed does not depend on which that is), for
    // all lanes of a warp.  -1: no more, or a wait ran out.
    auto take = [&](int k) -> int {
        const int q = k & 1;
        if (!__all_sync(0xffffffffu, tc_mbar_wait(&next_full[q], (k >> 1) & 1, abort_flag, st, 72))) return -1;
        const int index = __shfl_sync(0xffffffffu, next[q], 0);
        if (lane == 0) tc_mbar_arrive(&next_free[q]);
        return index < total ? index : -1;
    };

    if (warp == 0) {                                        // hands the items out and streams X' and Y'
        if (lane == 0) {
            tc_prefetch_tmap(&map_q);
            tc_prefetch_tmap(&map_g);
            int t = 0;                                      // stages filled
            bool ok = true;
            for (int k = 0; ok; ++k) {
                const int q = k & 1;
                if (k == 1) ab_wait_for_rows();
                const int index = k == 0 ? (int)blockIdx.x : (int)(gridDim.x + atomicAdd(w.taken, 1u));
                if (k >= 2 && !tc_mbar_wait(&next_free[q], ((k >> 1) - 1) & 1, abort_flag, st, 73)) break;
                next[q] = index;
                tc_mbar_arrive(&next_full[q]);
                if (index >= total) break;
                const ab_item it = ab_decode<PARTS>(a, work, index);
                if (k == 0 && it.keys) ab_wait_for_rows();
                const CUtensorMap *mx = it.keys ? &map_q : &map_k, *my = it.keys ? &map_g : &map_v;
                int sh = it.keys ? it.head * grp : it.head / grp, s = PARTS ? it.skip : 0;          // streamed head and tile of it
                if (PARTS && it.keys && it.n > 0) sh += s / it.per_head, s %= it.per_head;
                for (int i = 0; i < it.n; ++i, ++t) {
                    const int stage = t % Z::STAGES;
                    if (!tc_mbar_wait(&empty[stage], ((t / Z::STAGES) & 1) ^ 1, abort_flag, st, 61)) {
                        ok = false;
                        break;
                    }
                    const int r = (it.first + s) * AB_N;
                    uint8_t* to = ring + stage * 2 * Z::STEP;
                    tc_mbar_expect_tx(&full[stage], 2 * Z::STEP + (it.keys ? (TWICE ? 3 : 2) * AB_N * 4 : 0));
#pragma unroll
                    for (int b = 0; b < Z::BLOCKS; ++b) {
                        tc_tma_load_3d(to + b * (AB_N * 128), mx, &full[stage], b * 64, sh, r);
                        tc_tma_load_3d(to + Z::STEP + b * (AB_N * 128), my, &full[stage], b * 64, sh, r);
                    }
                    if (it.keys) {
                        float* rows = sRow + stage * 3 * AB_N;
                        tc_bulk_load(rows, w.neg_lse + (int64_t)sh * w.padded + r, &full[stage], AB_N * 4);
                        tc_bulk_load(rows + AB_N, w.d + (int64_t)sh * w.padded + r, &full[stage], AB_N * 4);
                        if (TWICE) tc_bulk_load(rows + 2 * AB_N, w.norm + (int64_t)sh * w.padded + r, &full[stage], AB_N * 4);
                    }
                    if (TWICE && !(i & 1)) continue;
                    if (++s == it.per_head) s = 0, ++sh;
                }
            }
            if (*abort_flag)
                for (int i = t > Z::STAGES ? t - Z::STAGES : 0; i < t; ++i) ab_drain(&full[i % Z::STAGES], (i / Z::STAGES) & 1);
        }
    } else if (warp == 2) {                                 // X and Y of the next item, as soon as these are not read any more
        int c = 0;                                          // walks so far
        for (int k = 0;; ++k) {
            const int index = take(k);
            if (index < 0) break;
            const ab_item it = ab_decode<PARTS>(a, work, index);
            if (it.n <= 0) continue;
            if (c > 0 && !__all_sync(0xffffffffu, tc_mbar_wait(own_free, (c - 1) & 1, abort_flag, st, 69))) break;
            if (lane == 0) {
                const CUtensorMap *mx = it.keys ? &map_k : &map_q, *my = it.keys ? &map_v : &map_g;
                tc_mbar_expect_tx(own_full, 2 * Z::OWN);
#pragma unroll
                for (int b = 0; b < Z::BLOCKS; ++b)
#pragma unroll
                    for (int h = 0; h < AB_M / AB_N; ++h) {
                        const int at = b * (AB_M * 128) + h * (AB_N * 128);
                        tc_tma_load_3d(sX + at, mx, own_full, b * 64, it.head, it.row0 + h * AB_N);
                        tc_tma_load_3d(sY + at, my, own_full, b * 64, it.head, it.row0 + h * AB_N);
                    }
            }
            __syncwarp();
            ++c;
        }
        if (lane == 0 && *abort_flag && c > 0) ab_drain(own_full, (c - 1) & 1);
    } else if (warp == 1) {
        if (tc_elect_one()) {
        // (one elected lane waits and issues)
        const uint32_t idesc_s = tc_idesc_f16(AB_M, AB_N, 0, 0), idesc_a = tc_idesc_f16(AB_M, HD, 0, 1);
        const uint64_t xd = tc_smem_desc(tc_smem_u32(sX), 16, 1024), yd = tc_smem_desc(tc_smem_u32(sY), 16, 1024);
        const uint32_t ring_at = tc_smem_u32(ring);
        auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
            const bool ok = tc_mbar_wait(bar, parity, abort_flag, st, site);
            tc_fence_after_sync();
            return ok;
        };
        int g0 = 0, c = 0, cq = 0;                              // steps (= stages), walks, walks of queries before this item
        // A walk.  Keys: X and Y from shared memory.  Queries: from TMEM, where they have room; that halves the operand bytes of S
        // and T, which shared memory's bandwidth bounds (48 cycles a product with both operands there, 32 with one).
        auto walk = [&](auto of_keys, const int n) -> bool {
            constexpr bool KEYS = decltype(of_keys)::value;
            auto scores = [&](int g) {                          // S = X X'^T and T = Y Y'^T of one step
                const uint32_t at = ring_at + (g % Z::STAGES) * 2 * Z::STEP, d = tmem + Z::SLOT + (g % Z::SLOTS) * (2 * AB_N);
                const uint64_t xs = tc_smem_desc(at, 16, 1024), ys = tc_smem_desc(at + Z::STEP, 16, 1024);
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    const uint32_t ao = ((kk >> 2) * (AB_M * 128) + (kk & 3) * 32) >> 4, bo = ((kk >> 2) * (AB_N * 128) + (kk & 3) * 32) >> 4;
                    if (KEYS) tc_mma_f16(d, xd + ao, xs + bo, idesc_s, kk != 0);
                    else tc_mma_f16_ts(d, tmem + Z::X + kk * 8, xs + bo, idesc_s, kk != 0);
                }
                if (Z::CUT) tc_mma_commit(&s_full[g % Z::SLOTS]);
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    const uint32_t ao = ((kk >> 2) * (AB_M * 128) + (kk & 3) * 32) >> 4, bo = ((kk >> 2) * (AB_N * 128) + (kk & 3) * 32) >> 4;
                    if (KEYS) tc_mma_f16(d + AB_N, yd + ao, ys + bo, idesc_s, kk != 0);
                    else tc_mma_f16_ts(d + AB_N, tmem + Z::Y + kk * 8, ys + bo, idesc_s, kk != 0);
                }
                tc_mma_commit(&(Z::CUT ? t_full : s_full)[g % Z::SLOTS]);
            };
            bool ok = wait(KEYS ? own_full : a_ready, (KEYS ? c : cq) & 1, 62);
            if (!KEYS && ok) tc_mbar_arrive(own_free);             // the softmax has moved them to TMEM
            for (int i = 0; i < Z::SLOTS && i < n && ok; ++i) {
                ok = wait(&full[(g0 + i) % Z::STAGES], ((g0 + i) / Z::STAGES) & 1, 63);
                if (ok) scores(g0 + i);
            }
            if (KEYS && ok && n <= Z::SLOTS) tc_mma_commit(own_free);   // (X and Y have been read when these products are done)
            for (int i = 0; i < n && ok; ++i) {
                const int g = g0 + i;
                const uint32_t at = ring_at + (g % Z::STAGES) * 2 * Z::STEP, p = tmem + Z::SLOT + (g % Z::SLOTS) * (2 * AB_N);
                const uint64_t xs = tc_smem_desc(at, AB_N * 128, 1024), ys = tc_smem_desc(at + Z::STEP, AB_N * 128, 1024);
                // the accumulators take the step, half by half where it is cut; its stage is free then
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (Z::CUT || h == 0) ok = ok && wait(&p_full[(g % Z::SLOTS) * 2 + h], (g / Z::SLOTS) & 1, 64);
                    if (ok && h == 0 && i == 0 && c > 0) ok = wait(acc_free, (c - 1) & 1, 70);
                    if (!ok) break;
                    if (KEYS) {
#pragma unroll
                        for (int kk = 2 * h; kk < 2 * h + 2; ++kk)
                            tc_mma_f16_ts(tmem + Z::ACC1, p + kk * 8, ys + (uint32_t)(kk * 2048 >> 4), idesc_a, (i > 0 || kk > 0) ? 1u : 0u);
                    }
#pragma unroll
                    for (int kk = 2 * h; kk < 2 * h + 2; ++kk)
                        tc_mma_f16_ts(tmem, p + AB_N + kk * 8, xs + (uint32_t)(kk * 2048 >> 4), idesc_a, (i > 0 || kk > 0) ? 1u : 0u);
                }
                if (!ok) break;
                tc_mma_commit(&empty[g % Z::STAGES]);
                if (i + Z::SLOTS < n) {
                    // (the tensor core runs one thread's products in their order: the slot has been read by then)
                    const int h = g + Z::SLOTS;
                    ok = wait(&full[h % Z::STAGES], (h / Z::STAGES) & 1, 65);
                    if (ok) scores(h);
                    if (KEYS && ok && i + Z::SLOTS == n - 1) tc_mma_commit(own_free);
                }
            }
            if (ok) tc_mma_commit(done);
            return ok;
        };
        for (int k = 0;; ++k) {
            if (!tc_mbar_wait(&next_full[k & 1], (k >> 1) & 1, abort_flag, st, 72)) break;
            const int index = next[k & 1];
            tc_mbar_arrive(&next_free[k & 1]);
            if (index >= total) break;
            const ab_item it = ab_decode<PARTS>(a, work, index);
            if (it.n <= 0) continue;
            if (!(it.keys ? walk(std::true_type(), it.n) : walk(std::false_type(), it.n))) break;
            g0 += it.n;
            ++c;
            cq += !it.keys;
        }
        }
    } else if (warp >= 4) {
        const int group = (warp - 4) >> 2;                      // two warpgroups take the steps in turn
        const int r = (warp & 3) * 32 + lane;                   // row of the tile == TMEM lane
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        // A hidden column's score is the infinity that the scale turns into -infinity, so that exp2 makes it a zero.  (A scale of
        // zero, times that, would be NaN: 2^-120 in its place moves no exponent, since f16 operands' scores are below 2^40.)
        const float sl = a.scale == 0.f ? 0x1p-120f : a.scale * AB_LOG2E;
        const uint32_t hidden = sl < 0.f ? 0x7f800000u : 0xff800000u;
        const uint64_t sl2 = at_pack2(sl, sl);
        ab_wait_for_rows();
        int g0 = 0, c = 0;
        bool of_keys_before = false;                            // the last walk was one of keys
        // Queries: the first warpgroup moves X, the second Y, from shared memory (a row is 16-byte pieces, swizzled by its number) to
        // TMEM.  `count`: the walk that they belong to.
        auto own = [&](int count) {
            // their place was the second accumulator of a walk of keys: both warpgroups have to have read it
            if (of_keys_before && !__all_sync(0xffffffffu, tc_mbar_wait(acc_free, (count - 1) & 1, abort_flag, st, 74))) return false;
            of_keys_before = false;
            tc_fence_after_sync();
            if (!__all_sync(0xffffffffu, tc_mbar_wait(own_full, count & 1, abort_flag, st, 71))) return false;
            const uint8_t* from = group ? sY : sX;
#pragma unroll
            for (int h = 0; h < HD / 64; ++h) {
                uint32_t v[32];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const uint4 x = *reinterpret_cast<const uint4*>(from + h * (AB_M * 128) + r * 128 + ((q ^ (r & 7)) * 16));
                    v[4 * q] = x.x, v[4 * q + 1] = x.y, v[4 * q + 2] = x.z, v[4 * q + 3] = x.w;
                }
                tc_tmem_st32(lanes + (group ? Z::Y : Z::X) + h * 32, v);
            }
            tc_tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) tc_mbar_arrive(a_ready);
            return true;
        };
        // What an item needs of its rows, asked for while the item before it ends.  A key's shift follows from its |V| and the largest
        // |dO| and |D| of the queries that see it: this lane's share of those that all keys of its warp see, and those of the first
        // query that its own key sees.  A query's follows from its |dO| and |D| and the largest |V| of the keys that it sees: this lane's
        // share of those that all queries of its warp see, and that of the last key that its own query sees.  And of a query 14 - lse / ln 2.
        struct ab_known { float most_g, most_d, most_v, g, d, v, nl; };
        auto ask = [&](const ab_item& it) {
            ab_known v = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, -INFINITY};
            const int kvh = it.keys ? it.head : it.head / grp;
            if (it.keys) {
                // Per head: queries own, own + 32, ... up to a block's end (own: the first that this lane's key sees), then whole
                // blocks; 32 of either at a time, four loads ahead of the arithmetic.
                const int rows = w.block >> w.q_log;
                long long own = 0, edge = 0;                    // (unmasked: all blocks)
                int block = 0, singles = 0;
                if (a.causal) {
                    const long long behind = (long long)it.row0 + (warp & 3) * 32 + 32 - a.causal_delta;      // queries from here on: all keys of the warp
                    const int from = behind < 0 ? 0 : behind > a.q_len ? a.q_len : (int)behind;
                    block = (from + rows - 1) / rows;
                    edge = block * rows < a.q_len ? block * rows : a.q_len;
                    singles = 1 + (int)((edge - from + 31) / 32);
                    own = behind - 32 + lane;
                }
                const int per_head = singles + (w.q_blocks - block + 31) / 32;
                int64_t head = (int64_t)kvh * grp;
                const int64_t head_end = head + grp;
                int c = 0;
#pragma unroll 1
                while (head < head_end) {
                    float2 m[4];
                    bool of_own[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        m[k] = make_float2(0.f, 0.f);
                        of_own[k] = c == 0 && singles;
                        if (head >= head_end) continue;
                        if (c < singles) {
                            const long long q = own + 32 * c;
                            if (q >= 0 && q < edge) m[k] = make_float2(w.norm[head * w.padded + q], w.d[head * w.padded + q]);
                        } else if (block + (c - singles) * 32 + lane < w.q_blocks) {
                            m[k] = w.most_q[head * w.q_blocks + block + (c - singles) * 32 + lane];
                        }
                        if (++c == per_head) c = 0, ++head;
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float d = fabsf(m[k].y) <= 3.0e38f ? fabsf(m[k].y) : 0.f;
                        if (of_own[k]) v.g = fmaxf(v.g, m[k].x), v.d = fmaxf(v.d, d);
                        else v.most_g = fmaxf(v.most_g, m[k].x), v.most_d = fmaxf(v.most_d, d);
                    }
                }
                if (it.row0 + r < a.kv_len) v.v = w.norm_v[(int64_t)kvh * a.kv_len + it.row0 + r];
            } else {
                const float *norms = w.norm_v + (int64_t)kvh * a.kv_len, *of_blocks = w.most_v + (int64_t)kvh * w.k_blocks;
                if (it.row0 + r < a.q_len) {
                    const int64_t at = (int64_t)it.head * w.padded + it.row0 + r;
                    v.nl = w.neg_lse[at];
                    v.d = w.d[at];
                    v.g = w.norm[at];
                }
                int blocks = w.k_blocks, edge = 0, single = 0;  // whole blocks that all queries of the warp see, then single keys
                if (a.causal) {
                    const long long first = (long long)it.row0 + (warp & 3) * 32 + 1 + a.causal_delta, own = first - 1 + lane;
                    if (own >= 0 && own < a.kv_len) v.v = norms[own];
                    if (first < a.kv_len) {
                        edge = first < 0 ? 0 : (int)first;
                        blocks = edge / (w.block >> w.k_log);
                        single = blocks * (w.block >> w.k_log);
                    }
                }
#pragma unroll 2
                for (int i = lane; i < blocks || single + i < edge; i += 32) {
                    const float x = i < blocks ? of_blocks[i] : 0.f, y = single + i < edge ? norms[single + i] : 0.f;
                    v.most_v = fmaxf(v.most_v, fmaxf(x, y));
                }
            }
            return v;
        };
        auto of_warp = [&](float x) {
#pragma unroll
            for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
            return x;
        };
        // Of this lane's value and those of the lanes behind it.
        auto of_later = [&](float x) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) x = fmaxf(x, __shfl_down_sync(0xffffffffu, x, o));
            return x;
        };
        // ... and those of the lanes before it.
        auto of_earlier = [&](float x) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) x = fmaxf(x, __shfl_up_sync(0xffffffffu, x, o));
            return x;
        };
        // Columns [32 h, 32 h + 32) of T: a difference of T and D within the rounding of their sums, 2^-22 of |dO| |V| of that query and
        // that key, is none: a query that sees one key has no gradient.  (Where there are more keys than a step's, others' gradients are far
        // above that.)  `near`: 2^-22 of this row's norm; `norms_v`: |V| of the keys, where the columns are keys.
        auto settle = [&](auto of_keys, uint32_t (&t)[32], const float4* rows, const float* norms_v, int h, float d, float near) {
            constexpr bool KEYS = decltype(of_keys)::value;
            const float* of_row = reinterpret_cast<const float*>(rows) + 32 * h;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                const float dj = KEYS ? of_row[AB_N + j] : d, norm = KEYS ? of_row[2 * AB_N + j] : 32 * h + j < a.kv_len ? norms_v[32 * h + j] : 0.f;
                if (fabsf(__uint_as_float(t[j]) - dj) <= near * norm) t[j] = __float_as_uint(dj);
            }
        };
        ab_known known = {};
        // One item: its steps, then its results.  `index` becomes the next item's.
        auto walk = [&](auto of_keys, const ab_item& it, int k, int& index) -> bool {
            constexpr bool KEYS = decltype(of_keys)::value;
            const int row = it.row0 + r;
            const float row_nl = known.nl, row_d = known.d;
            float most_g = known.g, most_v = known.v, most_d = fabsf(row_d);
            if (KEYS) most_g = fmaxf(of_warp(known.most_g), of_later(known.g)), most_d = fmaxf(of_warp(known.most_d), of_later(known.d));
            else most_v = fmaxf(of_warp(known.most_v), of_earlier(known.v));
            const float shrink = ab_shrink(most_g * most_v + most_d);
            const float near = (KEYS ? most_v : most_g) * 0x1p-22f;
            const float* norms_v = w.norm_v + (int64_t)(KEYS ? it.head : it.head / grp) * a.kv_len;
            const uint64_t shrink2 = at_pack2(shrink, shrink);
            const uint64_t row_nl2 = at_pack2(row_nl, row_nl), row_d2 = at_pack2(-row_d, -row_d);
            const int last = it.first + it.per_head;
            const int pace = TWICE ? 1 : 2;                           // streamed tiles from one of my steps to the next
            int s = (PARTS ? it.skip : 0) + ((g0 & 1) != group && pace == 2 ? 1 : 0);        // streamed tile of the step
            if (KEYS && it.n > 0 && s >= it.per_head) s = PARTS ? s % it.per_head : 0;
            s += it.first;
            for (int i = (g0 & 1) != group ? 1 : 0; i < it.n; i += 2) {
                const int g = g0 + i;
                const uint32_t slot = lanes + Z::SLOT + (g % Z::SLOTS) * (2 * AB_N);
                const int s0 = s * AB_N;                        // first streamed row of the step
                s += pace;
                const bool rest = TWICE && (i & 1);
                if (KEYS)
                    while (s >= last) s -= it.per_head;
                // columns [lo, hi) of this row are visible
                int lo = 0, hi = AB_N;
                bool masked = false;
                if (KEYS) {
                    if (a.causal && (long long)it.row0 + AB_M - 1 > (long long)s0 + a.causal_delta) {
                        const long long l = (long long)row - a.causal_delta - s0;
                        lo = l < 0 ? 0 : l > AB_N ? AB_N : (int)l;
                        masked = true;
                    }
                } else {
                    if (s0 + AB_N > a.kv_len || (a.causal && (long long)s0 + AB_N - 1 > (long long)it.row0 + a.causal_delta)) {
                        long long h = (long long)a.kv_len - s0;
                        if (a.causal && (long long)row + a.causal_delta + 1 - s0 < h) h = (long long)row + a.causal_delta + 1 - s0;
                        hi = h < 0 ? 0 : h > AB_N ? AB_N : (int)h;
                        masked = true;
                    }
                }
                // Half of the columns at a time.  Cut: P needs S alone, so that T may still be in the making; the sums over the first half
                // are made while the second one is worked on.  (Row values are asked for early: shared memory is busy with operands.)
                const float4* rows = reinterpret_cast<const float4*>(sRow + (g % Z::STAGES) * 3 * AB_N);
                float4 nl[8], dd[8];
                bool there = true;
                if (KEYS) {
                    there = tc_mbar_wait(&full[g % Z::STAGES], (g / Z::STAGES) & 1, abort_flag, st, 68);        // (the copies into sRow)
                    if (Z::CUT) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) nl[j] = rows[j];
                    }
                }
                there = there && tc_mbar_wait(&s_full[g % Z::SLOTS], (g / Z::SLOTS) & 1, abort_flag, st, 66);
                if (!__all_sync(0xffffffffu, there)) return false;
                tc_fence_after_sync();
                if constexpr (Z::CUT) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t s[32], t[32], half16[16];
                        tc_tmem_ld32(slot + 32 * h, s);
                        if (KEYS) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) dd[j] = rows[AB_N / 4 + 8 * h + j];
                        }
                        tc_tmem_ld_wait();
                        if (masked) {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (32 * h + j < lo || 32 * h + j >= hi) s[j] = hidden;
                        }
                        float p[32];
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            uint64_t nl2 = row_nl2;
                            if (KEYS) nl2 = (j & 2) ? at_pack2(nl[j >> 2].z, nl[j >> 2].w) : at_pack2(nl[j >> 2].x, nl[j >> 2].y);
                            float x0, x1;
                            at_unpack2(at_fma2(at_pack2(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), sl2, nl2), x0, x1);
                            p[j] = at_ex2(x0);
                            p[j + 1] = at_ex2(x1);
                            const __half2 hp = ab_pack<TWICE>(p[j], p[j + 1], rest);
                            half16[j >> 1] = *reinterpret_cast<const uint32_t*>(&hp);
                        }
                        // (over columns that this thread has read)
                        if (KEYS) tc_tmem_st16(slot + 16 * h, half16);
                        if (h == 0) {
                            if (!__all_sync(0xffffffffu, tc_mbar_wait(&t_full[g % Z::SLOTS], (g / Z::SLOTS) & 1, abort_flag, st, 75))) return false;
                            tc_fence_after_sync();
                        }
                        tc_tmem_ld32(slot + AB_N + 32 * h, t);
                        if (KEYS && h == 0) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) nl[j] = rows[8 + j];
                        }
                        tc_tmem_ld_wait();
                        if (TWICE && a.kv_len <= AB_N) settle(of_keys, t, rows, norms_v, h, row_d, near);
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            uint64_t d2 = row_d2;
                            if (KEYS) d2 = (j & 2) ? at_pack2(-dd[j >> 2].z, -dd[j >> 2].w) : at_pack2(-dd[j >> 2].x, -dd[j >> 2].y);
                            float y0, y1;
                            const uint64_t diff = at_add2(at_pack2(__uint_as_float(t[j]), __uint_as_float(t[j + 1])), d2);
                            at_unpack2(at_mul2(at_mul2(diff, shrink2), at_pack2(p[j], p[j + 1])), y0, y1);
                            const __half2 hs = ab_pack<TWICE>(y0, y1, rest);
                            half16[j >> 1] = *reinterpret_cast<const uint32_t*>(&hs);
                        }
                        tc_tmem_st16(slot + AB_N + 16 * h, half16);
                        tc_tmem_st_wait();
                        tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) tc_mbar_arrive(&p_full[(g % Z::SLOTS) * 2 + h]);
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t s[32], t[32], p16[16], s16[16];
                        tc_tmem_ld32(slot + 32 * h, s);
                        tc_tmem_ld32(slot + AB_N + 32 * h, t);
                        tc_tmem_ld_wait();
                        if (masked) {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (32 * h + j < lo || 32 * h + j >= hi) s[j] = hidden;
                        }
                        if (TWICE && a.kv_len <= AB_N) settle(of_keys, t, rows, norms_v, h, row_d, near);
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            uint64_t nl2 = row_nl2, d2 = row_d2;
                            if (KEYS) {
                                if (j % 4 == 0) nl[0] = rows[8 * h + j / 4], dd[0] = rows[AB_N / 4 + 8 * h + j / 4];
                                nl2 = (j & 2) ? at_pack2(nl[0].z, nl[0].w) : at_pack2(nl[0].x, nl[0].y);
                                d2 = (j & 2) ? at_pack2(-dd[0].z, -dd[0].w) : at_pack2(-dd[0].x, -dd[0].y);
                            }
                            float x0, x1, y0, y1;
                            at_unpack2(at_fma2(at_pack2(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), sl2, nl2), x0, x1);
                            const float p0 = at_ex2(x0), p1 = at_ex2(x1);
                            const uint64_t diff = at_add2(at_pack2(__uint_as_float(t[j]), __uint_as_float(t[j + 1])), d2);
                            at_unpack2(at_mul2(at_mul2(diff, shrink2), at_pack2(p0, p1)), y0, y1);
                            const __half2 hp = ab_pack<TWICE>(p0, p1, rest), hs = ab_pack<TWICE>(y0, y1, rest);
                            p16[j >> 1] = *reinterpret_cast<const uint32_t*>(&hp);
                            s16[j >> 1] = *reinterpret_cast<const uint32_t*>(&hs);
                        }
                        if (KEYS) tc_tmem_st16(slot + 16 * h, p16);
                        tc_tmem_st16(slot + AB_N + 16 * h, s16);
                    }
                    tc_tmem_st_wait();
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) tc_mbar_arrive(&p_full[(g % Z::SLOTS) * 2]);
                }
            }
            index = take(k + 1);
            ab_item then = it;
            if (index >= 0) {
                then = ab_decode<PARTS>(a, work, index);
                known = ask(then);
            }
            if (it.n > 0) {
                if (!__all_sync(0xffffffffu, tc_mbar_wait(done, c & 1, abort_flag, st, 67))) return false;
                tc_fence_after_sync();
            }
            // Every product of this item has been made.  If the next one is of queries too, its X and Y go to TMEM before the results
            // are read, so that its first scores are made meanwhile.
            if (!KEYS && index >= 0 && then.n > 0 && !own(c + (it.n > 0))) return false;
            // results: keys: the first warpgroup dK, the second dV; queries: half of the columns of dQ each
            const int row_end = KEYS ? a.dk_row0 + a.dk_rows : a.dq_row0 + a.dq_rows, warp_row = it.row0 + (warp & 3) * 32;
            const bool store = *abort_flag == 0;
            const float back = 0x1p-14f;
            const bool of_v = KEYS && group == 1;
            const int want = KEYS ? (of_v ? a.want & KTB_ATTN_DV : a.want & KTB_ATTN_DK) : a.want & KTB_ATTN_DQ;
            const int64_t row_stride = !KEYS ? a.dq_row : of_v ? a.dv_row : a.dk_row;
            const int64_t off = (int64_t)warp_row * row_stride + (!KEYS ? a.dq_off + (int64_t)it.head * a.dq_head
                                                                   : of_v ? a.dv_off + (int64_t)it.head * a.dv_head
                                                                          : a.dk_off + (int64_t)it.head * a.dk_head);
            float* sum = nullptr;                               // a part's sums stay f32
            if (PARTS && (KEYS ? work.key_parts : work.query_parts) > 1) {
                const int row_here = row - (KEYS ? a.dk_row0 : a.dq_row0), head_here = it.head - (KEYS ? a.dk_head0 : a.dq_head0);
                sum = (!KEYS ? work.part_q : of_v ? work.part_v : work.part_k) +
                      (((int64_t)it.part * (KEYS ? a.dk_rows : a.dq_rows) + row_here) * (KEYS ? a.dk_heads : a.dq_heads) + head_here) * HD + (KEYS ? 0 : group * (HD / 2));
            }
            const float factor = of_v ? back : a.scale * (back / shrink);
            constexpr int COLS = KEYS ? HD : HD / 2;
            const int col0 = KEYS ? 0 : group * (HD / 2);
            __half* dst = reinterpret_cast<__half*>(a.arena) + off + col0;
            const uint32_t from = lanes + (of_v ? Z::ACC1 : 0) + col0;
#pragma unroll
            for (int x = 0; x < COLS; x += 32) {
                uint32_t v[32];
                if (it.n > 0) {                                 // (the same for the whole warp)
                    tc_tmem_ld32(from + x, v);
                    tc_tmem_ld_wait();
                    if (x + 32 == COLS) {                       // all read: the next item may sum
                        tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) tc_mbar_arrive(acc_free);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = 0;
                }
                if (PARTS && sum) {
                    if (store && want && row < row_end) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            *reinterpret_cast<float4*>(sum + x + j) = make_float4(__uint_as_float(v[j]) * factor, __uint_as_float(v[j + 1]) * factor,
                                                                                 __uint_as_float(v[j + 2]) * factor, __uint_as_float(v[j + 3]) * factor);
                    }
                    __syncwarp();                               // (the next load takes the whole warp)
                } else if (want) {                              // (the same for the whole warp)
                    uint32_t o[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const __half2 h = __floats2half2_rn(__uint_as_float(v[2 * j]) * factor, __uint_as_float(v[2 * j + 1]) * factor);
                        o[j] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                    tc_store_rows(sOut + (warp - 4) * 2048, o, dst + x, row_stride, store ? row_end - warp_row : 0);
                }
            }
            return true;
        };
        int index = take(0);
        if (index >= 0) known = ask(ab_decode<PARTS>(a, work, index));
        bool keys_before = true;                                // the item before has not moved this one's X and Y
        for (int k = 0; index >= 0; ++k) {
            const ab_item it = ab_decode<PARTS>(a, work, index);
            if (!it.keys && keys_before && it.n > 0 && !own(c)) break;
            keys_before = it.keys;
            if (it.n > 0) of_keys_before = it.keys;
            if (!(it.keys ? walk(std::true_type(), it, k, index) : walk(std::false_type(), it, k, index))) break;
            g0 += it.n;
            c += it.n > 0;
        }
        tc_fence_before_sync();
    }
    __syncthreads();
    if (warp == 1) tc_tmem_dealloc(tmem, 512);
}

// Joins the parts of cut walks: sums in the order of the parts, rounded once.  Eight columns of a row to a thread.
struct ab_joined {
    const float* part;
    int64_t off, row, head;        // where the result goes
    int rows, heads, row0, head0, parts;
};

template <int HD>
__global__ void __launch_bounds__(256) ktb_attention_join_kernel(__half* arena, const ab_joined q, const ab_joined k, const ab_joined v) {
    const ab_joined t = blockIdx.y == 0 ? q : blockIdx.y == 1 ? k : v;
    const int64_t all = (int64_t)t.rows * t.heads * (HD / 8), at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t.parts < 2 || at >= all) return;
    float s[8] = {};
    for (int p = 0; p < t.parts; ++p) {
        const float4* from = reinterpret_cast<const float4*>(t.part + (p * all + at) * 8);
        const float4 x = from[0], y = from[1];
        s[0] += x.x, s[1] += x.y, s[2] += x.z, s[3] += x.w, s[4] += y.x, s[5] += y.y, s[6] += y.z, s[7] += y.w;
    }
    uint4 o;
    __half2* h = reinterpret_cast<__half2*>(&o);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(s[2 * i], s[2 * i + 1]);
    const int64_t r = at / (HD / 8);
    *reinterpret_cast<uint4*>(arena + t.off + (t.row0 + r / t.heads) * t.row + (t.head0 + r % t.heads) * t.head + (at % (HD / 8)) * 8) = o;
}

// Tensor [rows][heads][HD] in boxes of 64 rows x 64 columns of one head.
static bool ab_map(CUtensorMap* m, const ktb_attn_bwd_args& a, int64_t off, int64_t rows, int64_t heads, int64_t row, int64_t head) {
    const uint64_t dims[3] = {(uint64_t)a.head_dim, (uint64_t)heads, (uint64_t)rows};
    const uint64_t str[2] = {(uint64_t)head * 2, (uint64_t)row * 2};
    const uint32_t box[3] = {64, 1, AB_N};
    return tc_make_map_f16(m, reinterpret_cast<__half*>(a.arena) + off, 3, dims, str, box);
}

static int64_t ab_padded(const ktb_attn_bwd_args& a) { return ((int64_t)a.q_len + AB_N - 1) / AB_N * AB_N; }

// Neighbouring heads that a block of the rows kernel takes (a power of two, eight at most), and the rows of it.
static int ab_heads_log(int heads) { return heads >= 8 ? 3 : heads >= 4 ? 2 : heads >= 2 ? 1 : 0; }
static int64_t ab_row_blocks(int64_t rows, int heads, int block) { return (rows + (block >> ab_heads_log(heads)) - 1) / (block >> ab_heads_log(heads)); }
// Rows of heads to a block: few, where blocks of many would leave SMs idle (197 positions of 12 heads with their gradients 14.4 us,
// with 64 rows to a block 12.6; 1000 queries over 2777 keys of 32 / 8 heads 114.7, 116.0).
static int ab_block(const ktb_attn_bwd_args& a) { return (int64_t)a.q_len * a.heads + (int64_t)a.kv_len * (a.heads / a.kv_group) <= 16384 ? 64 : 256; }

static int64_t ab_up(int64_t bytes) { return (bytes + 255) / 256 * 256; }
// A counter; per query and head three floats, per key and key head one; per block of queries and head two, per block of keys and key
// head one ...
static int64_t ab_rows_bytes(const ktb_attn_bwd_args& a) {
    const int kv_heads = a.heads / a.kv_group;
    return ab_up(256 + 4 * (int64_t)a.heads * (3 * ab_padded(a) + 2 * ab_row_blocks(ab_padded(a), a.heads, ab_block(a))) +
                 4 * (int64_t)kv_heads * (ab_row_blocks(a.kv_len, kv_heads, ab_block(a)) + a.kv_len));
}
// ... and, of walks that are cut, the parts' sums.
static int64_t ab_part_bytes(const ktb_attn_bwd_args& a, bool keys) {
    const int parts = keys ? a.key_parts : a.query_parts;
    return parts < 2 ? 0 : ab_up(4 * (int64_t)parts * a.head_dim * (keys ? (int64_t)a.dk_rows * a.dk_heads : (int64_t)a.dq_rows * a.dq_heads));
}

extern "C" int64_t ktb_attention_bwd_scratch_bytes(const ktb_attn_bwd_args* args) {
    if (!args || args->kv_group < 1 || args->heads < args->kv_group || args->q_len < 1 || args->kv_len < 1) return 0;
    int64_t n = ab_rows_bytes(*args);
    if (args->want & KTB_ATTN_DQ) n += ab_part_bytes(*args, false);
    if (args->want & (KTB_ATTN_DK | KTB_ATTN_DV)) n += 2 * ab_part_bytes(*args, true);
    return n;
}

template <int HD>
static int ab_run(ktb_ctx* ctx, const ktb_attn_bwd_args& a) {
    const int kv_heads = a.heads / a.kv_group;
    ab_scratch w;
    w.padded = ab_padded(a);
    w.q_log = ab_heads_log(a.heads);
    w.k_log = ab_heads_log(kv_heads);
    w.block = ab_block(a);
    w.q_blocks = (int)ab_row_blocks(w.padded, a.heads, w.block);
    w.k_blocks = (int)ab_row_blocks(a.kv_len, kv_heads, w.block);
    const int64_t row_blocks = (int64_t)w.q_blocks * ((a.heads + (1 << w.q_log) - 1) >> w.q_log) + (int64_t)w.k_blocks * ((kv_heads + (1 << w.k_log) - 1) >> w.k_log);
    if (row_blocks > 0x7fffffff) return ktb_fail(ctx, KTB_E_UNSUPPORTED, "attention_bwd", "too many rows");
    w.taken = reinterpret_cast<unsigned*>(a.dev_scratch);
    w.neg_lse = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(a.dev_scratch) + 256);
    w.d = w.neg_lse + (int64_t)a.heads * w.padded;
    w.norm = w.d + (int64_t)a.heads * w.padded;
    w.most_q = reinterpret_cast<float2*>(w.norm + (int64_t)a.heads * w.padded);
    w.most_v = reinterpret_cast<float*>(w.most_q + (int64_t)a.heads * w.q_blocks);
    w.norm_v = w.most_v + (int64_t)kv_heads * w.k_blocks;
    CUtensorMap mq, mk, mv, mg;
    if (!ab_map(&mq, a, a.q_off, a.q_len, a.heads, a.q_row, a.q_head) || !ab_map(&mg, a, a.do_off, a.q_len, a.heads, a.do_row, a.do_head) ||
        !ab_map(&mk, a, a.k_off, a.kv_len, kv_heads, a.k_row, a.k_head) || !ab_map(&mv, a, a.v_off, a.kv_len, kv_heads, a.v_row, a.v_head))
        return ktb_fail(ctx, KTB_E_CUDA, "attention_bwd", "cuTensorMapEncodeTiled failed");
    const bool keys = (a.want & (KTB_ATTN_DK | KTB_ATTN_DV)) && a.dk_rows > 0 && a.dk_heads > 0;
    const bool queries = (a.want & KTB_ATTN_DQ) && a.dq_rows > 0 && a.dq_heads > 0;
    const bool join_q = queries && a.query_parts > 1, join_k = keys && a.key_parts > 1;
    const int64_t nq = join_q ? (int64_t)a.dq_rows * a.dq_heads : 0, nk = join_k ? (int64_t)a.dk_rows * a.dk_heads : 0;
    const int64_t blocks = ((nq > nk ? nq : nk) * (HD / 8) + 255) / 256;
    if (blocks > 0x7fffffff) return ktb_fail(ctx, KTB_E_UNSUPPORTED, "attention_bwd", "too many rows in parts");
    (w.block == 64 ? ktb_attention_rows_kernel<HD, 64> : ktb_attention_rows_kernel<HD, 256>)<<<(unsigned)row_blocks, 256, 0, ctx->stream>>>(a, w);
    KTB_CHECK_LAUNCH(ctx, "ktb_attention_rows_kernel");
    static bool attr_set[KTB_MAX_DEVICES] = {};     // the attribute is per device
    if (!attr_set[ctx->device & (KTB_MAX_DEVICES - 1)]) {
        KTB_CUDA(ctx, cudaFuncSetAttribute(ktb_attention_bwd_kernel<HD, 0>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ab_shape<HD>::SMEM));
        KTB_CUDA(ctx, cudaFuncSetAttribute(ktb_attention_bwd_kernel<HD, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ab_shape<HD>::SMEM));
        KTB_CUDA(ctx, cudaFuncSetAttribute(ktb_attention_bwd_kernel<HD, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ab_shape<HD>::SMEM));
        attr_set[ctx->device & (KTB_MAX_DEVICES - 1)] = true;
    }
    ab_work work;
    work.key_tiles = keys ? (a.dk_rows + AB_M - 1) / AB_M : 0;
    work.key_heads = keys ? a.dk_heads : 0;
    work.query_tiles = queries ? (a.dq_rows + AB_M - 1) / AB_M : 0;
    work.query_heads = queries ? a.dq_heads : 0;
    work.key_parts = a.key_parts > 1 ? a.key_parts : 1;
    work.query_parts = a.query_parts > 1 ? a.query_parts : 1;
    work.twice = a.twice;
    const long long items = (long long)work.key_tiles * work.key_heads * work.key_parts + (long long)work.query_tiles * work.query_heads * work.query_parts;
    uint8_t* parts = reinterpret_cast<uint8_t*>(a.dev_scratch) + ab_rows_bytes(a);
    work.part_q = reinterpret_cast<float*>(parts);
    parts += (a.want & KTB_ATTN_DQ) ? ab_part_bytes(a, false) : 0;
    work.part_k = reinterpret_cast<float*>(parts);
    work.part_v = reinterpret_cast<float*>(parts + ab_part_bytes(a, true));
    if (items == 0) return KTB_OK;
    if (items > 0x3fffffff) return ktb_fail(ctx, KTB_E_UNSUPPORTED, "attention_bwd", "too many tiles");
    work.by_head = items >= 16ll * ctx->sm_count;
    const int grid = items < ctx->sm_count ? (int)items : ctx->sm_count;
    // It sets up, and fetches what does not come from the kernel before it, while that one ends.
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(384);
    config.dynamicSmemBytes = ab_shape<HD>::SMEM;
    config.stream = ctx->stream;
    config.attrs = &early;
    config.numAttrs = 1;
    // (not cutting is a kernel of its own: finding a part cost the others up to 9 %)
    auto kernel = a.twice ? ktb_attention_bwd_kernel<HD, 2> : work.key_parts > 1 || work.query_parts > 1 ? ktb_attention_bwd_kernel<HD, 1> : ktb_attention_bwd_kernel<HD, 0>;
    KTB_CUDA(ctx, cudaLaunchKernelEx(&config, kernel, mq, mk, mv, mg, a, w, work, ctx->dev_status));
    if (join_q || join_k) {
        KTB_CHECK_LAUNCH(ctx, "ktb_attention_bwd_kernel");
        ab_joined q = {work.part_q, a.dq_off, a.dq_row, a.dq_head, a.dq_rows, a.dq_heads, a.dq_row0, a.dq_head0, join_q ? work.query_parts : 0};
        ab_joined k = {work.part_k, a.dk_off, a.dk_row, a.dk_head, a.dk_rows, a.dk_heads, a.dk_row0, a.dk_head0, join_k && (a.want & KTB_ATTN_DK) ? work.key_parts : 0};
        ab_joined v = {work.part_v, a.dv_off, a.dv_row, a.dv_head, a.dk_rows, a.dk_heads, a.dk_row0, a.dk_head0, join_k && (a.want & KTB_ATTN_DV) ? work.key_parts : 0};
        ktb_attention_join_kernel<HD><<<dim3((unsigned)blocks, 3), 256, 0, ctx->stream>>>(reinterpret_cast<__half*>(a.arena), q, k, v);
        KTB_CHECK_LAUNCH(ctx, "ktb_attention_join_kernel");
        return KTB_OK;
    }
    KTB_CHECK_LAUNCH(ctx, "ktb_attention_bwd_kernel");
    return KTB_OK;
}

extern "C" int ktb_launch_attention_bwd(ktb_ctx* ctx, const ktb_attn_bwd_args* args) {
    if (!ctx || !args) return KTB_E_ARG;
    const ktb_attn_bwd_args& a = *args;
    const char* me = "attention_bwd";
    if (a.head_dim != 64 && a.head_dim != 128) return ktb_fail(ctx, KTB_E_UNSUPPORTED, me, "head_dim must be 64 or 128");
    if (a.q_len < 0 || a.kv_len < 0 || a.heads < 0 || a.kv_group < 1 || a.heads % a.kv_group)
        return ktb_fail(ctx, KTB_E_ARG, me, "lengths, heads or kv_group");
    if (a.key_parts < 0 || a.key_parts > 64 || a.query_parts < 0 || a.query_parts > 64 || a.twice < 0 || a.twice > 1) return ktb_fail(ctx, KTB_E_ARG, me, "parts of a walk");
    if ((a.want & ~7) || a.want == 0) return ktb_fail(ctx, KTB_E_ARG, me, "which gradients are wanted");
    if (a.q_len == 0 || a.kv_len == 0 || a.heads == 0) return ktb_fail(ctx, KTB_E_UNSUPPORTED, me, "no queries, keys or heads");
    if (a.q_len > (1 << 30) || a.kv_len > (1 << 30) || a.heads > 65535 * 32) return ktb_fail(ctx, KTB_E_UNSUPPORTED, me, "lengths or heads");
    if (((int64_t)a.q_len + AB_N - 1) / AB_N * a.kv_group > (1 << 28)) return ktb_fail(ctx, KTB_E_UNSUPPORTED, me, "too many steps of a tile of keys");
    if (!(fabs((double)a.scale) * a.head_dim * 65504.0 * 65504.0 <= 1.0e38))     // (scores of f16 operands, times 1 / ln 2)
        return ktb_fail(ctx, KTB_E_ARG, me, "scores must be finite");
    const int kv_heads = a.heads / a.kv_group;
    if (a.want & KTB_ATTN_DQ)
        if (a.dq_row0 < 0 || a.dq_rows < 0 || a.dq_rows > a.q_len - a.dq_row0 || a.dq_head0 < 0 || a.dq_heads < 0 || a.dq_heads > a.heads - a.dq_head0)
            return ktb_fail(ctx, KTB_E_ARG, me, "rows or heads of dQ outside the tensors");
    if (a.want & (KTB_ATTN_DK | KTB_ATTN_DV))
        if (a.dk_row0 < 0 || a.dk_rows < 0 || a.dk_rows > a.kv_len - a.dk_row0 || a.dk_head0 < 0 || a.dk_heads < 0 || a.dk_heads > kv_heads - a.dk_head0)
            return ktb_fail(ctx, KTB_E_ARG, me, "rows or heads of dK and dV outside the tensors");
    const int64_t all = a.q_off | a.k_off | a.v_off | a.o_off | a.do_off | a.q_row | a.q_head | a.k_row | a.k_head | a.v_row | a.v_head |
                        a.o_row | a.o_head | a.do_row | a.do_head | ((a.want & KTB_ATTN_DQ) ? a.dq_off | a.dq_row | a.dq_head : 0) |
                        ((a.want & KTB_ATTN_DK) ? a.dk_off | a.dk_row | a.dk_head : 0) | ((a.want & KTB_ATTN_DV) ? a.dv_off | a.dv_row | a.dv_head : 0);
    if ((all & 7) || (reinterpret_cast<uintptr_t>(a.arena) & 15))
        return ktb_fail(ctx, KTB_E_UNSUPPORTED, me, "strides and offsets must be multiples of 8 elements");
    if (!a.dev_scratch || (reinterpret_cast<uintptr_t>(a.dev_scratch) & 255) || a.scratch_bytes < ktb_attention_bwd_scratch_bytes(args))
        return ktb_fail(ctx, KTB_E_ARG, me, "scratch too small or not on a 256-byte boundary");
    return a.head_dim == 64 ? ab_run<64>(ctx, a) : ab_run<128>(ctx, a);
}
