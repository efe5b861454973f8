// Rotary positions: pairs (x, y) of every head turned by the angle of the token's position,
//   x' = x cos - y sin,  y' = y cos + x sin   (backwards: with -sin),
// with cos and sin gathered from tables by position, products and sums rounded to f32 one by one (what the KTIR
// program says), the result rounded once; the elements of a head behind the pairs are copied.  It takes over the op
// sequence indirect ktdp.load of two table rows, arith.mulf / subf / addf on broadcast tiles, ktdp.store, which the
// reference dispatches op by op (ktir_cpu/ops/memory_ops.py:867-915, ktir_cpu/dialects/arith_ops.py:49-59).
//
// HBM bounds it: every element is read and written once (8192 tokens of 72 heads of 128, f16: 52 us, 5.9 TB/s; a token is a
// launch, 4 us).  A thread owns VEC pairs (16 bytes of x and of y, or of
// adjacent pairs), or as many bytes behind the pairs, of up to HEADS heads of one token, so that it reads its table entries
// once for all of them and has their loads in flight together; the position -> table -> product chain is entered after they
// have been issued (asked for first, the position holds them up: 8192 tokens of 72 heads, 128 wide, 52 us -> 66).  What turns
// and what is copied is loaded by the same instructions, since lanes of one warp do either (f32, 4001 tokens of 40 heads, 96
// wide, half of it turned: 36 us in branches of their own, 27 together).
#include "tc_common.cuh"

template <typename T> static __device__ __forceinline__ float ro_up(T v);
template <> __device__ __forceinline__ float ro_up<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float ro_up<float>(float v) { return v; }
template <typename T> static __device__ __forceinline__ T ro_down(float v);
template <> __device__ __forceinline__ __half ro_down<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float ro_down<float>(float v) { return v; }

template <typename T, int N> struct __align__(sizeof(T) * N) ro_vec { T e[N]; };

// Copies `n` elements; `bytes` (a power of two up to 16) is what both addresses and the length are multiples of.
template <typename T>
static __device__ __forceinline__ void ro_copy16(const T* src, T* dst, int bytes, int n) {
    if (bytes == 16) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
    else if (bytes == 8) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(src);
    else if (bytes == 4) *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(src);
    else for (int i = 0; i < n; ++i) dst[i] = src[i];
}

// ADJ: x and y are neighbours (interleaved pairs), VEC pairs in one vector; else VEC pairs are a vector of x and one of
// y (VEC = 1: any pair stride).  ONE: a single item.  REST: something is copied.
template <typename T, bool ADJ, int VEC, int HEADS, bool ONE, bool REST>
__global__ void __launch_bounds__(256)
ktb_rotary_kernel(const ktb_rotary_args a, int64_t token0, uint32_t n_threads, uint32_t slots, uint32_t chunks, uint32_t turn_chunks,
                  int heads_total, int rest_bytes, int table_vec, ktb_status* st) {
    typedef ro_vec<T, ADJ ? 2 * VEC : VEC> V;
    const uint32_t g = blockIdx.x * 256u + threadIdx.x;
    if (g >= n_threads) return;
    const uint32_t c = g % chunks, r = g / chunks;
    const uint32_t slot = r % slots;
    const int64_t token = token0 + r / slots;
    const int64_t item = ONE ? 0 : token / a.tokens;
    const int tok = (int)(token - item * a.tokens);
    const int64_t* off = ONE ? a.first : a.dev_item_offsets + item * (1 + 2 * a.n_tensors);
    T* arena = reinterpret_cast<T*>(a.arena);
    const bool turn = !REST || c < turn_chunks;
    // where this thread's elements of the heads slot, slot + slots, ... (counted over all tensors) lie
    const int per = turn ? VEC : rest_bytes >= 4 ? rest_bytes / (int)sizeof(T) : 1;
    const int j0 = (int)(turn ? c : c - turn_chunks) * per;
    const T* src[HEADS];
    T* dst[HEADS];
    int which[HEADS];
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
        int h = (int)(slot + k * slots), t = 0;
        which[k] = -1;
        src[k] = arena;
        dst[k] = arena;
        if (h < heads_total) {
            while (h >= a.t[t].heads) h -= a.t[t++].heads;
            if (turn || j0 < a.t[t].rest) which[k] = t;
            src[k] += off[1 + 2 * t] + tok * a.t[t].in_token + h * a.t[t].in_head + (turn ? (int64_t)j0 * (ADJ ? 2 : a.pair_stride) : a.t[t].in_rest + j0);
            dst[k] += off[2 + 2 * t] + tok * a.t[t].out_token + h * a.t[t].out_head + (turn ? (int64_t)j0 * (ADJ ? 2 : a.pair_stride) : a.t[t].out_rest + j0);
        }
    }
    if (REST && !turn && rest_bytes != (int)sizeof(V)) {          // no vectors like those of the pairs
#pragma unroll
        for (int k = 0; k < HEADS; ++k)
            if (which[k] >= 0) ro_copy16(src[k], dst[k], rest_bytes, per);
        return;
    }
    V x[HEADS], y[HEADS];                         // (ADJ: x holds the pairs, y is not used)
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
        if (which[k] < 0) continue;
        x[k] = *reinterpret_cast<const V*>(src[k]);
        if (!ADJ && turn) y[k] = *reinterpret_cast<const V*>(src[k] + a.t[which[k]].in_partner);
    }
    if (turn) {
        const int64_t pe = off[0] + tok * a.pos_stride;
        int64_t pos = a.idx_dtype == KTB_I64 ? reinterpret_cast<const int64_t*>(a.arena)[pe] : (int64_t)reinterpret_cast<const int32_t*>(a.arena)[pe];
        if (pos < 0) {
            if (atomicExch(&st->negative_index, 1) == 0) st->bad_index_value = (int32_t)pos;
            pos = 0;
        }
        float cs[VEC], sn[VEC];
        const float* table = reinterpret_cast<const float*>(a.arena);
#pragma unroll
        for (int which_table = 0; which_table < 2; ++which_table) {
            float* into = which_table ? sn : cs;
            const int64_t end = which_table ? a.sin_end : a.cos_end, base = which_table ? a.sin_off : a.cos_off;
            // (a position far behind the table reads zeros like any address past the end; the product cannot pass 63 bits)
            const int64_t at = pos < (int64_t)1 << 40 ? base + pos * a.table_stride + j0 : end;
            if (VEC % 4 == 0 && table_vec && at + VEC <= end) {
#pragma unroll
                for (int i = 0; i < VEC / 4; ++i) {
                    const float4 f = reinterpret_cast<const float4*>(table + at)[i];
                    into[4 * i] = f.x, into[4 * i + 1] = f.y, into[4 * i + 2] = f.z, into[4 * i + 3] = f.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) into[i] = at + i < end ? table[at + i] : 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) sn[i] = a.inverse ? -sn[i] : sn[i];         // (a sign does not change a rounding)
#pragma unroll
        for (int k = 0; k < HEADS; ++k) {
            if (which[k] < 0) continue;
            V v;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float fx = ro_up<T>(x[k].e[ADJ ? 2 * i : i]), fy = ro_up<T>(ADJ ? x[k].e[ADJ ? 2 * i + 1 : 0] : y[k].e[i]);
                const T rx = ro_down<T>(__fsub_rn(__fmul_rn(fx, cs[i]), __fmul_rn(fy, sn[i])));
                const T ry = ro_down<T>(__fadd_rn(__fmul_rn(fy, cs[i]), __fmul_rn(fx, sn[i])));
                x[k].e[ADJ ? 2 * i : i] = rx;
                if (ADJ) x[k].e[ADJ ? 2 * i + 1 : 0] = ry;
                else v.e[i] = ry;
            }
            *reinterpret_cast<V*>(dst[k]) = x[k];
            if (!ADJ) *reinterpret_cast<V*>(dst[k] + a.t[which[k]].out_partner) = v;
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < HEADS; ++k)
        if (which[k] >= 0) *reinterpret_cast<V*>(dst[k]) = x[k];
}

// The same where the halves of a head, or what is behind them, start off the 16-byte boundaries that the head itself is on (27
// pairs of f16, say): a thread owns 16 bytes of a head, wherever they fall.  What they are turned with is in the same bytes
// (adjacent pairs) or n elements on or back: two neighbouring vectors, shifted into one; a vector that holds the end of the first
// half needs both.  Table values are kept for several heads of the token, whose own bytes are on their way together; the rest
// of a head comes from L1.  4096 tokens of 40 heads, 128 wide, 54 turned: halves 61 us element by element, 39 so; adjacent pairs
// 45 in 4-byte vectors, 23 so.  Instructions bound it (f32, with half as many elements to 16 bytes, moves twice the bytes).
// VEC elements from `shift` on in the 2 * VEC of lo and hi.
template <typename T, typename V>
static __device__ __forceinline__ V ro_shift(const V& lo, const V& hi, int shift) {
    uint32_t w[9];
    const uint32_t* l = reinterpret_cast<const uint32_t*>(&lo);
    const uint32_t* h = reinterpret_cast<const uint32_t*>(&hi);
    const int words = sizeof(T) == 2 ? shift >> 1 : shift;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = l[i], w[4 + i] = h[i];
    w[8] = 0;
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = words & 2 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = words & 1 ? w[i + 1] : w[i];
    V y;
    uint32_t* to = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = sizeof(T) == 2 && (shift & 1) ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
    return y;
}

// (nothing that is read is written: later loads need not wait for earlier stores)
template <typename V>
static __device__ __forceinline__ V ro_ldg(const void* p) { const uint4 q = __ldg(reinterpret_cast<const uint4*>(p)); return *reinterpret_cast<const V*>(&q); }

template <typename T, bool ADJ>
__global__ void __launch_bounds__(256, 4)
ktb_rotary_rows_kernel(const ktb_rotary_args a, int64_t token0, uint32_t n_threads, uint32_t slots, int row_vecs, int heads_total, ktb_status* st) {
    constexpr int VEC = 16 / (int)sizeof(T), HEADS = 4, PAIRS = ADJ ? VEC / 2 : VEC;
    typedef ro_vec<T, VEC> V;
    const uint32_t g = blockIdx.x * 256u + threadIdx.x;
    if (g >= n_threads) return;
    const uint32_t c = g % (uint32_t)row_vecs, r = g / (uint32_t)row_vecs;
    const int64_t token = token0 + r / slots;
    const int64_t item = a.n_items == 1 ? 0 : token / a.tokens;
    const int tok = (int)(token - item * a.tokens);
    const int64_t* off = a.n_items == 1 ? a.first : a.dev_item_offsets + item * (1 + 2 * a.n_tensors);
    T* arena = reinterpret_cast<T*>(a.arena);
    const int n = a.pairs, e0 = (int)c * VEC;
    const bool turn = e0 < 2 * n;
    // !ADJ: the other half's elements start at `other`; `split`: those of this vector's later elements n back, in front of the head
    const bool split = !ADJ && e0 < n && e0 + VEC > n;
    const int other = e0 < n ? e0 + n : e0 - n, shift = other % VEC, end = (row_vecs - 1) * VEC;
    uint64_t cs[VEC / 2], sn[VEC / 2];                   // factors of elements 2i and 2i + 1, and of their partners
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) cs[i] = sn[i] = 0;
    // (gone round once: a thread has four heads, or one.  Without the loop the compiler starts on the tables before the heads' own loads,
    // with more spilled: 23 us -> 29 for adjacent pairs, 39 -> 42 for halves.)
#pragma unroll 1
    for (int first = (int)(r % slots); first < heads_total; first += HEADS * (int)slots) {
        V x[HEADS];
        const T* src[HEADS];
        T* dst[HEADS];
#pragma unroll
        for (int k = 0; k < HEADS; ++k) {
            int h = first + k * (int)slots, t = 0;
            dst[k] = nullptr;
            src[k] = arena;
            if (h >= heads_total) continue;
            while (h >= a.t[t].heads) h -= a.t[t++].heads;
            src[k] = arena + off[1 + 2 * t] + tok * a.t[t].in_token + h * a.t[t].in_head;
            dst[k] = arena + off[2 + 2 * t] + tok * a.t[t].out_token + h * a.t[t].out_head + e0;
            x[k] = *reinterpret_cast<const V*>(src[k] + e0);
        }
        if (turn) {
            const int64_t pe = off[0] + tok * a.pos_stride;
            int64_t pos = a.idx_dtype == KTB_I64 ? reinterpret_cast<const int64_t*>(a.arena)[pe] : (int64_t)reinterpret_cast<const int32_t*>(a.arena)[pe];
            if (pos < 0) {
                if (atomicExch(&st->negative_index, 1) == 0) st->bad_index_value = (int32_t)pos;
                pos = 0;
            }
            const float* table = reinterpret_cast<const float*>(a.arena);
            const int64_t row = pos < (int64_t)1 << 40 ? pos * a.table_stride : (int64_t)1 << 61;
            // entries of pair j0 + i, or, from the other half on, of e - n (a row past the table's end is zeros, one across it in part)
            const int j0 = ADJ ? e0 / 2 : e0 < n ? e0 : e0 - n, wrap = ADJ || e0 >= n ? VEC : n - e0;
            const int64_t in_cos = a.cos_end - a.cos_off - row, in_sin = a.sin_end - a.sin_off - row;
            const float *cr = table + (in_cos > 0 ? a.cos_off + row : 0), *sr = table + (in_sin > 0 ? a.sin_off + row : 0);
            const int nc = in_cos < n ? in_cos < 0 ? 0 : (int)in_cos : n, ns = in_sin < n ? in_sin < 0 ? 0 : (int)in_sin : n;
            float c[PAIRS], s[PAIRS];
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                const int j = i < wrap ? j0 + i : i - wrap;
                c[i] = j < nc ? cr[j] : 0.f;
                s[i] = j < ns ? sr[j] : 0.f;
                if (a.inverse != (!ADJ && e0 + i < n)) s[i] = -s[i];         // (x' = x cos + y (-sin))
            }
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
                cs[i] = ADJ ? at_pack2(c[i], c[i]) : at_pack2(c[2 * i], c[2 * i + 1]);
                sn[i] = ADJ ? at_pack2(-s[i], s[i]) : at_pack2(s[2 * i], s[2 * i + 1]);
            }
        }
#pragma unroll
        for (int k = 0; k < HEADS; ++k) {
            if (!dst[k]) continue;
            V v = x[k], y = x[k];
            if (!ADJ && turn) {
                // (other lanes have loaded these; a second vector past the head holds nothing that is wanted)
                const int at = other - shift;
                const V lo = ro_ldg<V>(src[k] + at);
                y = shift ? ro_shift<T>(lo, at < end ? ro_ldg<V>(src[k] + at + VEC) : lo, shift) : lo;
                if (split) {
                    const V head = ro_ldg<V>(src[k]), back = ro_shift<T>(head, head, VEC - (n - e0));
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        if (e0 + i >= n) y.e[i] = back.e[i];
                }
            }
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
                // (two products at a time; their sums one by one, since a pair of them becomes an fma, which does not round the product)
                const uint64_t own = at_pack2(ro_up<T>(x[k].e[2 * i]), ro_up<T>(x[k].e[2 * i + 1]));
                const uint64_t partner = ADJ ? at_pack2(ro_up<T>(x[k].e[2 * i + 1]), ro_up<T>(x[k].e[2 * i])) : at_pack2(ro_up<T>(y.e[2 * i]), ro_up<T>(y.e[2 * i + 1]));
                float mc0, mc1, os0, os1;
                at_unpack2(at_mul2(own, cs[i]), mc0, mc1);
                at_unpack2(at_mul2(partner, sn[i]), os0, os1);
                if (e0 + 2 * i < 2 * n)                      // (behind the pairs: copied)
                    v.e[2 * i] = ro_down<T>(__fadd_rn(mc0, os0)), v.e[2 * i + 1] = ro_down<T>(__fadd_rn(mc1, os1));
            }
            *reinterpret_cast<V*>(dst[k]) = v;
        }
    }
}

template <typename T, bool ADJ>
static int launch_rotary_rows(ktb_ctx* ctx, const ktb_rotary_args& a, int heads_total, int row_vecs) {
    const int64_t tokens = a.n_items * a.tokens;
    // four heads to a thread where two waves of threads are left all the same
    uint32_t slots = (uint32_t)(heads_total + 3) / 4;
    if (tokens * slots * row_vecs < (int64_t)ctx->sm_count * 2048) slots = (uint32_t)heads_total;
    const int64_t per_token = (int64_t)slots * row_vecs;
    if (per_token > 1 << 30) return ktb_fail(ctx, KTB_E_UNSUPPORTED, "rotary", "more than 2^30 vectors per token");
    const int64_t step = ((int64_t)1 << 30) / per_token;
    for (int64_t t0 = 0; t0 < tokens; t0 += step) {
        const int64_t n = tokens - t0 < step ? tokens - t0 : step;
        const uint32_t threads = (uint32_t)(n * per_token);
        ktb_rotary_rows_kernel<T, ADJ><<<(threads + 255) / 256, 256, 0, ctx->stream>>>(a, t0, threads, slots, row_vecs, heads_total, ctx->dev_status);
        KTB_CHECK_LAUNCH(ctx, "ktb_rotary_rows_kernel");
    }
    return KTB_OK;
}

template <typename T, bool ADJ, int VEC>
static int launch_rotary(ktb_ctx* ctx, const ktb_rotary_args& a, int heads_total, int rest, int rest_bytes, int table_vec) {
    const int64_t tokens = a.n_items * a.tokens;
    const uint32_t turn = (uint32_t)(a.pairs / VEC), per = rest_bytes >= 4 ? rest_bytes / (int)sizeof(T) : 1;
    const uint32_t chunks = turn + (uint32_t)((rest + (int)per - 1) / (int)per);
    // Four heads to a thread where two waves of threads are left all the same.
    const bool four = tokens * ((heads_total + 3) / 4) * chunks >= (int64_t)ctx->sm_count * 2048 * 2;
    const uint32_t slots = four ? (uint32_t)(heads_total + 3) / 4 : (uint32_t)heads_total;
    const int64_t per_token = (int64_t)slots * chunks;
    if (per_token > 1 << 30) return ktb_fail(ctx, KTB_E_UNSUPPORTED, "rotary", "more than 2^30 vectors per token");
    const int64_t step = ((int64_t)1 << 30) / per_token;          // tokens per launch: thread numbers stay within 32 bits
    for (int64_t t0 = 0; t0 < tokens; t0 += step) {
        const int64_t n = tokens - t0 < step ? tokens - t0 : step;
        const uint32_t threads = (uint32_t)(n * per_token);
        const bool one = a.n_items == 1;
        auto kernel = rest ? (four ? (one ? ktb_rotary_kernel<T, ADJ, VEC, 4, true, true> : ktb_rotary_kernel<T, ADJ, VEC, 4, false, true>)
                                   : (one ? ktb_rotary_kernel<T, ADJ, VEC, 1, true, true> : ktb_rotary_kernel<T, ADJ, VEC, 1, false, true>))
                           : (four ? (one ? ktb_rotary_kernel<T, ADJ, VEC, 4, true, false> : ktb_rotary_kernel<T, ADJ, VEC, 4, false, false>)
                                   : (one ? ktb_rotary_kernel<T, ADJ, VEC, 1, true, false> : ktb_rotary_kernel<T, ADJ, VEC, 1, false, false>));
        kernel<<<(threads + 255) / 256, 256, 0, ctx->stream>>>(a, t0, threads, slots, chunks, turn, heads_total, rest_bytes, table_vec, ctx->dev_status);
        KTB_CHECK_LAUNCH(ctx, "ktb_rotary_kernel");
    }
    return KTB_OK;
}

extern "C" int ktb_launch_rotary(ktb_ctx* ctx, const ktb_rotary_args* args) {
    if (!ctx || !args) return KTB_E_ARG;
    const ktb_rotary_args& a = *args;
    if (a.n_tensors < 1 || a.n_tensors > KTB_ROTARY_TENSORS) return ktb_fail(ctx, KTB_E_ARG, "rotary", "number of tensors");
    if (a.dtype != KTB_F16 && a.dtype != KTB_F32) return ktb_fail(ctx, KTB_E_UNSUPPORTED, "rotary", "f16 or f32 tensors");
    if (a.idx_dtype != KTB_I32 && a.idx_dtype != KTB_I64) return ktb_fail(ctx, KTB_E_UNSUPPORTED, "rotary", "i32 or i64 positions");
    if (a.pairs <= 0 || a.pair_stride < 1 || a.tokens < 0 || a.n_items < 0 || a.table_stride < 0)
        return ktb_fail(ctx, KTB_E_ARG, "rotary", "pairs, strides and counts");
    if (a.align < 1 || (a.align & (a.align - 1))) return ktb_fail(ctx, KTB_E_ARG, "rotary", "align must be a power of two");
    if ((uintptr_t)a.arena & (a.idx_dtype == KTB_I64 ? 7 : 3)) return ktb_fail(ctx, KTB_E_ARG, "rotary", "arena off the boundaries of tables and positions");
    const int size = a.dtype == KTB_F16 ? 2 : 4;
    // the lowest set bit of `bits` divides every distance between the vectors of pairs, that of `rest_bits` those behind them
    const int64_t start = (int64_t)a.align | (int64_t)((uintptr_t)a.arena / size);
    int64_t heads_total = 0, bits = start, rest_bits = start;
    int rest = 0;
    bool adjacent = a.pair_stride == 2;
    for (int t = 0; t < a.n_tensors; ++t) {
        const ktb_rotary_tensor& x = a.t[t];
        if (x.heads < 0 || x.rest < 0 || x.in_partner < 1 || x.out_partner < 1) return ktb_fail(ctx, KTB_E_ARG, "rotary", "heads, rest or partner");
        heads_total += x.heads;
        rest = x.rest > rest ? x.rest : rest;
        const int64_t strides = x.in_token | x.in_head | x.out_token | x.out_head;
        bits |= strides;
        if (x.rest) rest_bits |= strides | x.in_rest | x.out_rest | x.rest;
        adjacent = adjacent && x.in_partner == 1 && x.out_partner == 1;
    }
    if (a.n_items == 0 || a.tokens == 0 || heads_total == 0) return KTB_OK;
    if (!a.dev_item_offsets) return ktb_fail(ctx, KTB_E_ARG, "rotary", "null item table");
    if (heads_total > 1 << 20) return ktb_fail(ctx, KTB_E_UNSUPPORTED, "rotary", "more than 2^20 heads");
    if (!adjacent)
        for (int t = 0; t < a.n_tensors; ++t) bits |= a.t[t].in_partner | a.t[t].out_partner;
    bits |= adjacent ? 2 * (int64_t)a.pairs : a.pairs;
    // A vector is as long as every address and distance allows, 16 bytes at most.
    int vec = (int)(bits & -bits);
    vec = vec * size > 16 || vec <= 0 ? 16 / size : vec;
    int rest_vec = (int)(rest_bits & -rest_bits);
    if (adjacent && vec < 2) adjacent = false;
    if (!adjacent && a.pair_stride != 1) vec = 1;
    const int rest_bytes = rest_vec * size > 16 || rest_vec <= 0 ? 16 : rest_vec * size;
    // Heads that are one run of 16-byte vectors, their halves or rests not.
    const int64_t dim = 2 * (int64_t)a.pairs + rest;
    bool whole = dim * size % 16 == 0 && (start & (16 / size - 1)) == 0 && (adjacent || a.pair_stride == 1);
    for (int t = 0; t < a.n_tensors; ++t) {
        const ktb_rotary_tensor& x = a.t[t];
        whole = whole && ((x.in_token | x.in_head | x.out_token | x.out_head) & (16 / size - 1)) == 0 && x.rest == rest &&
                (rest == 0 || (x.in_rest == 2 * a.pairs && x.out_rest == 2 * a.pairs)) && (adjacent || (x.in_partner == a.pairs && x.out_partner == a.pairs));
    }
    if (whole && (vec * size < 16 || (rest && rest_bytes < 16))) {
        const int row_vecs = (int)(dim * size / 16), H = (int)heads_total;
        if (a.dtype == KTB_F16) return adjacent ? launch_rotary_rows<__half, true>(ctx, a, H, row_vecs) : launch_rotary_rows<__half, false>(ctx, a, H, row_vecs);
        return adjacent ? launch_rotary_rows<float, true>(ctx, a, H, row_vecs) : launch_rotary_rows<float, false>(ctx, a, H, row_vecs);
    }
    const int table_vec = ((a.table_stride | a.cos_off | a.sin_off | (int64_t)((uintptr_t)a.arena / 4)) & 3) == 0;
    const int H = (int)heads_total;
    if (a.dtype == KTB_F16) {
        if (adjacent)
            return vec == 8 ? launch_rotary<__half, true, 4>(ctx, a, H, rest, rest_bytes, table_vec)
                 : vec == 4 ? launch_rotary<__half, true, 2>(ctx, a, H, rest, rest_bytes, table_vec)
                            : launch_rotary<__half, true, 1>(ctx, a, H, rest, rest_bytes, table_vec);
        return vec == 8 ? launch_rotary<__half, false, 8>(ctx, a, H, rest, rest_bytes, table_vec)
             : vec == 4 ? launch_rotary<__half, false, 4>(ctx, a, H, rest, rest_bytes, table_vec)
             : vec == 2 ? launch_rotary<__half, false, 2>(ctx, a, H, rest, rest_bytes, table_vec)
                        : launch_rotary<__half, false, 1>(ctx, a, H, rest, rest_bytes, table_vec);
    }
    if (adjacent)
        return vec == 4 ? launch_rotary<float, true, 2>(ctx, a, H, rest, rest_bytes, table_vec)
                        : launch_rotary<float, true, 1>(ctx, a, H, rest, rest_bytes, table_vec);
    return vec == 4 ? launch_rotary<float, false, 4>(ctx, a, H, rest, rest_bytes, table_vec)
         : vec == 2 ? launch_rotary<float, false, 2>(ctx, a, H, rest, rest_bytes, table_vec)
                    : launch_rotary<float, false, 1>(ctx, a, H, rest, rest_bytes, table_vec);
}
