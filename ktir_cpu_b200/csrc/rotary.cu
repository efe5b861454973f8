// Rotary positions: pairs (x, y) of every head turned by the angle of the token's position,
//   x' = x cos - y sin,  y' = y cos + x sin   (backwards: with -sin),
// with cos and sin gathered from tables by position, products and sums rounded to f32 one by one (what the KTIR
// program says), the result rounded once; the elements of a head behind the pairs are copied.  It takes over the op
// sequence indirect ktdp.load of two table rows, arith.mulf / subf / addf on broadcast tiles, ktdp.store, which the
// reference dispatches op by op (ktir_cpu/ops/memory_ops.py:867-915, ktir_cpu/dialects/arith_ops.py:49-59).
//
// HBM bounds it: every element is read and written once.  A thread owns VEC pairs (16 bytes of x and of y, or of
// adjacent pairs) of up to HEADS heads of one token, so that it reads its table entries once for all of them and has
// their loads in flight together; the position -> table -> product chain is entered after they have been issued.
#include "common.cuh"

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
// y (VEC = 1: any pair stride).
template <typename T, bool ADJ, int VEC, int HEADS>
__global__ void __launch_bounds__(256)
ktb_rotary_kernel(const ktb_rotary_args a, int64_t token0, uint32_t n_threads, uint32_t slots, uint32_t chunks, uint32_t turn_chunks,
                  int heads_total, int rest_bytes, int table_vec, ktb_status* st) {
    const uint32_t g = blockIdx.x * 256u + threadIdx.x;
    if (g >= n_threads) return;
    const uint32_t c = g % chunks, r = g / chunks;
    const uint32_t slot = r % slots;
    const int64_t token = token0 + r / slots;
    const int64_t item = token / a.tokens;
    const int tok = (int)(token - item * a.tokens);
    const int64_t* off = a.dev_item_offsets + item * (1 + 2 * a.n_tensors);
    T* arena = reinterpret_cast<T*>(a.arena);

    // the heads of this thread: slot, slot + slots, ... counted over all tensors
    const T* src[HEADS];
    T* dst[HEADS];
    int which[HEADS];
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
        int h = (int)(slot + k * slots), t = 0;
        which[k] = -1;
        if (h < heads_total) {
            while (h >= a.t[t].heads) h -= a.t[t++].heads;
            which[k] = t;
            src[k] = arena + off[1 + 2 * t] + tok * a.t[t].in_token + h * a.t[t].in_head;
            dst[k] = arena + off[2 + 2 * t] + tok * a.t[t].out_token + h * a.t[t].out_head;
        }
    }
    if (c >= turn_chunks) {                       // behind the pairs
        const int per = rest_bytes >= 4 ? rest_bytes / (int)sizeof(T) : 1;
        const int at = (int)(c - turn_chunks) * per;
#pragma unroll
        for (int k = 0; k < HEADS; ++k) {
            if (which[k] < 0) continue;
            const ktb_rotary_tensor& t = a.t[which[k]];
            if (at < t.rest) ro_copy16(src[k] + t.in_rest + at, dst[k] + t.out_rest + at, rest_bytes, per);
        }
        return;
    }
    const int j0 = (int)c * VEC;
    typedef ro_vec<T, ADJ ? 2 * VEC : VEC> V;
    V x[HEADS], y[HEADS];                         // (ADJ: x holds the pairs, y is not used)
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
        if (which[k] < 0) continue;
        const T* p = src[k] + (int64_t)j0 * (ADJ ? 2 : a.pair_stride);
        x[k] = *reinterpret_cast<const V*>(p);
        if (!ADJ) y[k] = *reinterpret_cast<const V*>(p + a.t[which[k]].in_partner);
    }
    const int64_t pe = off[0] + tok * a.pos_stride;
    int64_t pos = a.idx_dtype == KTB_I64 ? reinterpret_cast<const int64_t*>(a.arena)[pe]
                                         : (int64_t)reinterpret_cast<const int32_t*>(a.arena)[pe];
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
    if (a.inverse) {                              // (a sign does not change a rounding)
#pragma unroll
        for (int i = 0; i < VEC; ++i) sn[i] = -sn[i];
    }
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
        if (which[k] < 0) continue;
        V u, v;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float fx = ro_up<T>(x[k].e[ADJ ? 2 * i : i]), fy = ro_up<T>(ADJ ? x[k].e[ADJ ? 2 * i + 1 : 0] : y[k].e[i]);
            const T rx = ro_down<T>(__fsub_rn(__fmul_rn(fx, cs[i]), __fmul_rn(fy, sn[i])));
            const T ry = ro_down<T>(__fadd_rn(__fmul_rn(fy, cs[i]), __fmul_rn(fx, sn[i])));
            u.e[ADJ ? 2 * i : i] = rx;
            if (ADJ) u.e[ADJ ? 2 * i + 1 : 0] = ry;
            else v.e[i] = ry;
        }
        T* p = dst[k] + (int64_t)j0 * (ADJ ? 2 : a.pair_stride);
        *reinterpret_cast<V*>(p) = u;
        if (!ADJ) *reinterpret_cast<V*>(p + a.t[which[k]].out_partner) = v;
    }
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
        if (four)
            ktb_rotary_kernel<T, ADJ, VEC, 4><<<(threads + 255) / 256, 256, 0, ctx->stream>>>(a, t0, threads, slots, chunks, turn, heads_total, rest_bytes, table_vec, ctx->dev_status);
        else
            ktb_rotary_kernel<T, ADJ, VEC, 1><<<(threads + 255) / 256, 256, 0, ctx->stream>>>(a, t0, threads, slots, chunks, turn, heads_total, rest_bytes, table_vec, ctx->dev_status);
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
    const int table_vec = ((a.table_stride | a.cos_off | a.sin_off) & 3) == 0;
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
