// Softmax attention over long rows with modified scores, forward and backward (bf16, head_dim 32 / 64, shared key heads):
//     s = scale q.k     cap: s = cap tanh(s / cap)     bias: s -= slope_h sum_a |pos_q[i, a] - pos_k[j, a]|
//     visible (i, j):  doc_q[i] == doc_k[j] >= 0   and   j < max(prefix, i + Nk - Nq + 1)  when causal
//     p = softmax over the visible j      o = p v      (a row that sees nothing: o = 0, lse = -inf)
//     dv = p^T do    dp = do v^T    ds = p (dp - sum(do o)) (1 - tanh^2)    dq = scale ds k    dk = scale ds^T q
//
// Layout.  A wave owns 32 rows (queries, or keys in the dk / dv kernel) and multiplies with v_mfma_f32_32x32x16_bf16 so that every LANE owns one
// of them: S^T = K Q^T leaves lane = query and registers = keys, so row maximum, sum and rescale are lane-local (one exchange between the
// wave's halves), and the same registers, packed to bf16, are the right operand of the next product (O^T = V^T P^T): its contraction index
// may come in any order as long as both operands agree, and V^T fragments read from LDS with ds_read_b64_tr_b16 take the accumulator's
// order.  Scores never leave the registers.  Tiles of 64 keys go global -> LDS by DMA one tile ahead of the products, double-buffered, one
// barrier per tile.
//
// Masks by tiles.  With documents, a small launch leaves the smallest and largest document and the count of valid tokens of every 64-token tile; a
// workgroup tests 64 tiles at a time (one per lane, one ballot) and walks only tiles that some row of it may see.  Per wave a tile is skipped,
// whole (no test per score) or partial; in a partial one a lane holds what it sees as one bit per row of the tile.  Rows of up to 256 tokens are
// walked without tables (forward, 32 x 8 heads, one document a row: 128 tokens 9.9 us without and 12.4 with, 256 15.8 and 17.7, 512 43.9 and
// 43.7, there with several documents 69 and 55).  The row blocks of packed rows differ in length; where there are more than two of them for a
// CU, the launch also puts them in order, the longest first (8 x 12 heads of 1024 in five documents: forward 49 -> 41 us, backward 140 -> 110; one
// row of 8192 in twelve documents, 16 heads: backward 240 -> 200).
//
// Sums, maxima, lse and all products accumulate in fp32.  p is rounded to bf16 as an operand of the second product (at most 2^-8 of each weight,
// averaging over what is summed; its sum is taken before the rounding): o and dv are 0.0019 to 0.0026 from the 64-bit result, the most where few
// terms count, where 0.0017 is the rounding of the result itself.  (In two parts, like ds, all four results are at 0.0017, for 4 to 15 % more time
// of a step: 16 over 4 heads of 4095 tokens behind a prefix forward 100 -> 134 us, backward 376 -> 412; 8 x 12 heads of 1024 in five documents 41 ->
// 44 and 110 -> 114; 16 heads of 8192 with a distance 74 -> 82 and 200 -> 212; one query of 4097 keys 45 -> 47.)  ds goes into its product as two
// bf16 parts, and sum(do o) takes o with what its rounding left out: dq and dk are then 0.0017 to 0.0024 from the 64-bit gradient.  In one part they
// were 0.0024 to 0.0031 away (the terms of a sum that nearly cancel are rounded apart) for 8 to 18 % less time of the backward pass.  Scores are
// fp32: forward takes them up to 2^30 in size (the exponent's reference point is rounded like them), backward forms p from lse, off by |lse| 2^-23
// of its value (2^-9 at scores of 2^14).
//
// What bounds it: the arithmetic between the products.  At 16 heads of 4095 tokens behind a prefix a score costs 7 vector operations forward, 10 for
// dq, 11 for dk and dv; the vector pipe is busy 66 % and the matrix pipe 32 % of the forward pass (100 us, 690 TFLOP/s), 61 / 44 % for dq and
// 44 / 38 % for dk and dv (375 us together with their joining, 820 TFLOP/s counting the products that are made).  A distance of two axes takes
// the forward pass to 16 operations, padded rows counted (64 x 12 heads of 257 tokens, 52 us, 61 with lse and o's remainder: 55 / 13 %).  One query
// of many keys is bound by HBM: 16 x 12 heads of 4097 keys in 43 us, 4.7 TB/s; query heads that share keys read them again, out of L2 (16 over 4
// heads: 41.5 us for 67 MB of keys and values).
//
// Values that are not finite behind a mask: 0 * inf would reach the products, so in partial tiles the rows of the second product's left
// operand that hold such values are replaced by zeros in LDS and noted; a row that SEES one of them is NaN in full.
//
// No atomics on results: dq is owned by queries, dk / dv by keys (the scores are computed twice), split rows are joined in a fixed order.
#include "gemm_common.h"
#include "mirage_hip.h"

namespace {

constexpr float LOG2E_F = 1.4426950408889634f, LN2_F = 0.6931471805599453f;
constexpr int TT = 64;                        // tokens of a staged tile
constexpr int MAX_SPLITS = 64;
struct ModArgs {
    const bf16_t* q; const bf16_t* k; const bf16_t* v; bf16_t* o; bf16_t* o_rest; float* lse;
    long q_bs, q_rs, q_hs, k_bs, k_rs, k_hs, v_bs, v_rs, v_hs, o_bs, o_rs, o_hs;
    int B, H, Hk, G, Nq, Nk;                  // G = H / Hk
    float scale, cap;
    const float* slopes; const float* pos_q; const float* pos_k; int axes;
    const int* doc_q; const int* doc_k;
    const int4* tab_q; const int4* tab_k; int ntq, ntk;     // per tile {lowest, highest document, valid tokens}; null: every tile is looked at
    int causal; const int* prefix;
    const bf16_t* d_o; long do_bs, do_rs, do_hs;
    bf16_t* dq; bf16_t* dk; bf16_t* dv;
    long dq_bs, dq_rs, dq_hs, dk_bs, dk_rs, dk_hs, dv_bs, dv_rs, dv_hs;
    float* dsum;                              // [B, H, Nq] sum(do o)
    float* part; float* part_ml; int splits;  // split rows: [split][rows][HD] unnormalised, [split][rows][2] {max, sum}
    int nblk, abreast;                        // row blocks of the owner; do the heads' blocks start side by side
    const int* order;                         // [B][nblk]: the row blocks, longest first (null: causal order tells, or they are alike)
};

// byte offset of 16-byte chunk c of row r in a [TT][HD] bf16 tile; the XOR spreads the rows that one instruction reads over the banks
template <int HD> __device__ __forceinline__ int swz(int r) { return HD == 64 ? (r >> 1) & 7 : (r >> 2) & 3; }
template <int HD> __device__ __forceinline__ int toff(int r, int c) { return r * HD * 2 + ((c ^ swz<HD>(r)) << 4); }
__device__ __forceinline__ bf16x8 lds_read16(uint32_t addr, int byte_off) {
    typedef __attribute__((address_space(3))) bf16x8 lds_v;
    return *((lds_v*)(uintptr_t)addr + (byte_off >> 4));
}
// operand with the contraction along hd: lane -> row (lane & 31) of a block of 32, chunk 2 kk + (lane >> 5); one LDS address per kk, the block of
// rows is an immediate offset
template <int HD> struct RowFrag {
    uint32_t at[HD / 16];
    __device__ __forceinline__ void init(int lane) {
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) at[kk] = (uint32_t)toff<HD>(lane & 31, 2 * kk + (lane >> 5));
    }
    __device__ __forceinline__ bf16x8 read(uint32_t tile, int row0, int kk) const { return lds_read16(tile + at[kk], row0 * HD * 2); }
};
// operand with the contraction along the tile's rows in accumulator order (rows base + 0..3, base + 8..11, base = row0 + 4 (lane >> 5), row0 a multiple
// of 16), lane -> hd element 32 dj + (lane & 31)
template <int HD> struct ColFrag {
    uint32_t at[HD / 32][2];
    __device__ __forceinline__ void init(int lane) {
        const int i = lane & 15, r = 4 * (lane >> 5) + (i >> 2);
#pragma unroll
        for (int dj = 0; dj < HD / 32; ++dj) {
            const int d = dj * 32 + (lane & 16) + ((i & 3) << 2);
            at[dj][0] = (uint32_t)(toff<HD>(r, d >> 3) + ((d & 4) << 1));
            at[dj][1] = (uint32_t)(toff<HD>(r + 8, d >> 3) + ((d & 4) << 1));
        }
    }
    __device__ __forceinline__ bf16x8 read(uint32_t tile, int row0, int dj) const {
        const s16x4 a = lds_read_tr16_off(tile + at[dj][0], row0 * HD * 2), b = lds_read_tr16_off(tile + at[dj][1], row0 * HD * 2);
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};
__device__ __forceinline__ bf16x8 pack_half(const f32x16& s, int m) {
    const uint4 w = make_uint4(pack_bf2(s[8 * m], s[8 * m + 1]), pack_bf2(s[8 * m + 2], s[8 * m + 3]), pack_bf2(s[8 * m + 4], s[8 * m + 5]), pack_bf2(s[8 * m + 6], s[8 * m + 7]));
    return __builtin_bit_cast(bf16x8, w);
}
// what the rounding of s to bf16 (pack_half) left out, itself in bf16: a product with both parts sees s to 2^-17
__device__ __forceinline__ bf16x8 pack_rest(const f32x16& s, int m, const bf16x8& hi) {
    const uint4 h = __builtin_bit_cast(uint4, hi);
    const uint32_t w[4] = {h.x, h.y, h.z, h.w};
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = pack_bf2(s[8 * m + 2 * i] - __uint_as_float(w[i] << 16), s[8 * m + 2 * i + 1] - __uint_as_float(w[i] & 0xffff0000u));
    return __builtin_bit_cast(bf16x8, make_uint4(r[0], r[1], r[2], r[3]));
}
__device__ __forceinline__ f32x16 zero16() { f32x16 z; for (int i = 0; i < 16; ++i) z[i] = 0.f; return z; }
// the value of this lane and of its partner in the other half of the wave
__device__ __forceinline__ float2 halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// minimum / maximum over the wave, in registers: four DPP steps within 16 lanes, then the swaps of rows and of halves
template <bool MAX> __device__ __forceinline__ int pick(int a, int b) { return MAX ? max(a, b) : min(a, b); }
template <bool MAX> __device__ __forceinline__ int wave_pick(int v) {
    v = pick<MAX>(v, __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, true));      // quad_perm [1,0,3,2]
    v = pick<MAX>(v, __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, true));      // quad_perm [2,3,0,1]
    v = pick<MAX>(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xF, 0xF, true));     // row_half_mirror
    v = pick<MAX>(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xF, 0xF, true));     // row_mirror
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = pick<MAX>(r[0], r[1]);
    const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return pick<MAX>(h[0], h[1]);
}
__device__ __forceinline__ int wave_min_i(int v) { return wave_pick<false>(v); }
__device__ __forceinline__ int wave_max_i(int v) { return wave_pick<true>(v); }

// does any of the 8 bf16 values have an all-ones exponent
__device__ __forceinline__ bool not_finite(const uint4 w) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    const u16x2 a = __builtin_bit_cast(u16x2, w.x & 0x7fff7fffu), b = __builtin_bit_cast(u16x2, w.y & 0x7fff7fffu);
    const u16x2 c = __builtin_bit_cast(u16x2, w.z & 0x7fff7fffu), d = __builtin_bit_cast(u16x2, w.w & 0x7fff7fffu);
    const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(a, b), __builtin_elementwise_max(c, d));
    return m[0] >= 0x7f80 || m[1] >= 0x7f80;
}

// ---- staging: a tile goes global -> LDS by DMA, 1 KiB (64 chunks of 16 bytes, whole rows) an instruction; the swizzle is applied to the
// address a lane reads from.  Rows behind the last one repeat it.  NW waves share the blocks of a tile; a wave's are 2 NW apart in parity
// pairs, so that one offset register per parity serves all of them (the swizzle has a period of 16 rows).
template <int HD, int NW>
struct Dma {
    static constexpr int CPR = HD / 8, RPB = 64 / CPR, NB = TT / RPB, PER = NB / NW;      // rows per block, blocks per tile and per wave
    static constexpr int PAR = (HD == 64 && NW == 1) ? 2 : 1;
    uint32_t off[PAR];
    int rs2;
    __device__ __forceinline__ int block(int j, int wave) const {                          // j-th block of this wave
        if (NW == 1) return j;
        return HD == 64 ? (wave & 1) + 4 * (wave >> 1) + 2 * j : wave;
    }
    __device__ __forceinline__ void init(long rs, int lane, int wave) {
        rs2 = (int)rs * 2;
#pragma unroll
        for (int p = 0; p < PAR; ++p) {
            const int r = (PAR == 2 ? p : (HD == 64 ? wave & 1 : 0)) * RPB + lane / CPR;
            off[p] = (uint32_t)(r * rs2 + (((lane % CPR) ^ swz<HD>(r)) << 4));
        }
    }
    // rows row0 .. row0 + TT - 1 of `base` (uniform) into `lds`; n: rows there are
    __device__ __forceinline__ void fetch(const bf16_t* base, int row0, int n, const char* lds, int lane, int wave) const {
        const char* tile = reinterpret_cast<const char*>(base) + (long)row0 * rs2;
        const uint32_t dst = lds_addr(lds);
        if (row0 + TT <= n) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int b = block(j, wave), odd = HD == 64 ? b & 1 : 0;
                glds16_s(uniform_ptr(tile + (long)(b - odd) * RPB * rs2), off[PAR == 2 ? odd : 0], __builtin_amdgcn_readfirstlane(dst + b * 1024));
            }
        } else {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int b = block(j, wave), r = b * RPB + lane / CPR;
                const uint32_t o = (uint32_t)(min(r, n - 1 - row0) * rs2 + (((lane % CPR) ^ swz<HD>(r)) << 4));
                glds16_s(uniform_ptr(tile), o, __builtin_amdgcn_readfirstlane(dst + b * 1024));
            }
        }
    }
    // this wave's part of a landed tile: values that are not finite become zero, their rows are noted
    __device__ __forceinline__ void tidy(char* lds, unsigned long long* noted, int lane, int wave) const {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int b = block(j, wave);
            uint4* at = reinterpret_cast<uint4*>(lds + b * 1024 + lane * 16);
            if (not_finite(*at)) {
                *at = make_uint4(0, 0, 0, 0);
                atomicOr(noted, 1ull << (b * RPB + lane / CPR));
            }
        }
    }
};
__device__ __forceinline__ void dma_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// smallest / largest document and number of valid tokens of a tile whose tokens the wave's lanes hold
__device__ __forceinline__ int4 doc_range(int d) {
    return make_int4(wave_min_i(d < 0 ? 0x7fffffff : d), wave_max_i(d), __popcll(__builtin_amdgcn_ballot_w64(d >= 0)), 0);
}
// ... of every tile of every batch row: the queries' tiles, then the keys' (no tiles of queries where both sides are the same tokens)
__global__ __launch_bounds__(256) void doc_tiles_kernel(const int* __restrict__ doc_q, const int* __restrict__ doc_k, int4* __restrict__ tab_q, int4* __restrict__ tab_k,
                                                        int B, int Nq, int Nk, int ntq, int ntk) {
    int t = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const bool ofk = t >= B * ntq;
    if (ofk) t -= B * ntq;
    const int nt = ofk ? ntk : ntq, N = ofk ? Nk : Nq;
    if (t >= B * nt) return;
    const int b = t / nt, j = (t - b * nt) * TT + lane;
    const int4 e = doc_range(j < N ? (ofk ? doc_k : doc_q)[(long)b * N + j] : -1);
    if (lane == 0) (ofk ? tab_k : tab_q)[t] = e;
}

// Work of a launch: `heads` (batch, head) pairs of `per` row blocks each.  Workgroups are dispatched round-robin over the 8 dies; a die gets whole
// heads (where they divide by 8), so that a head's keys stay in its own L2.  abreast: all heads' first blocks start first; otherwise a head's blocks
// follow each other.
__device__ __forceinline__ void place(int id, int heads, int per, int abreast, int& head, int& blk) {
    const int dies = heads % 8 == 0 ? 8 : 1, mine = heads / dies;
    const int die = id % dies, idx = id / dies;
    if (abreast) { head = die * mine + idx % mine; blk = idx / mine; }
    else { head = die * mine + idx / per; blk = idx % per; }
}

// Tables and order of the row blocks in one launch, one workgroup per batch row: the tiles' ranges, the number of tiles that each block of `rows` rows
// will walk, and the blocks by that number, the longest first (equal ones in their place).  order_q: blocks of queries, order_k (may be null):
// of keys.  At 8192 tokens in 12 documents and 16 heads the blocks walk 5 to 18 tiles; dispatched as they come the last round ran half empty.
constexpr int ORDER_TILES = 512, ORDER_THREADS = 1024, ORDER_PARTS = 8;
struct OrderArgs { const int* doc_q; const int* doc_k; int4* tab_q; int4* tab_k; int* order_q; int* order_k; int Nq, Nk, ntq, ntk, rows, causal; const int* prefix; };
__device__ __forceinline__ void order_tiles(const int* __restrict__ doc, int N, int nt, int4* table, int4* __restrict__ out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    constexpr int W = ORDER_THREADS / 64;
    for (int t0 = wave; t0 < nt; t0 += 8 * W) {
        int d[8];                                                 // eight tiles of this wave requested at once
#pragma unroll
        for (int i = 0; i < 8; ++i) { const int j = (t0 + W * i) * TT + lane; d[i] = j < N ? doc[j] : -1; }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int t = t0 + W * i;
            const int4 e = doc_range(d[i]);
            if (t < nt && lane == 0) { table[t] = e; out[t] = e; }
        }
    }
}
__device__ __forceinline__ int part_sum(int v) { for (int o = 1; o < ORDER_PARTS; o <<= 1) v += __shfl_xor(v, o, 64); return v; }
__global__ __launch_bounds__(ORDER_THREADS) void doc_order_kernel(const OrderArgs a) {
    __shared__ int4 tq[ORDER_TILES], tk[ORDER_TILES];
    __shared__ int count[ORDER_TILES];
    const int b = blockIdx.x;
    const bool same = a.doc_q == a.doc_k && a.Nq == a.Nk;
    order_tiles(a.doc_k + (long)b * a.Nk, a.Nk, a.ntk, tk, a.tab_k + (long)b * a.ntk);
    if (!same) order_tiles(a.doc_q + (long)b * a.Nq, a.Nq, a.ntq, tq, a.tab_q + (long)b * a.ntq);
    const int off = a.Nk - a.Nq, pre = a.causal ? (a.prefix ? min(max(a.prefix[b], 0), a.Nk) : 0) : a.Nk;
    const bool alike = same && !a.causal;                         // keys are seen by as many tiles as queries see
    const int part = threadIdx.x % ORDER_PARTS;
    for (int side = 0; side < (a.order_k && !alike ? 2 : 1); ++side) {
        const int N = side ? a.Nk : a.Nq, nblk = (N + a.rows - 1) / a.rows, nts = side ? a.ntq : a.ntk;
        const int4* own = side || same ? tk : tq;
        const int4* other = !side || same ? tk : tq;
        __syncthreads();
        for (int i0 = 0; i0 < nblk; i0 += ORDER_THREADS / ORDER_PARTS) {
            const int i = i0 + threadIdx.x / ORDER_PARTS;
            int n = 0;
            if (i < nblk) {
                const int r0 = i * a.rows, r1 = min(r0 + a.rows, N) - 1;
                int lo = 0x7fffffff, hi = -1;
                for (int t = r0 / TT; t <= r1 / TT; ++t) { lo = min(lo, own[t].x); hi = max(hi, own[t].y); }
                const int edge = side ? (r0 < pre ? 0 : r0 - off) : max(pre, min(r1 + off + 1, a.Nk));
                for (int t = part; t < nts; t += ORDER_PARTS) n += other[t].x <= hi && other[t].y >= lo && (side ? t * TT + TT > edge : t * TT < edge);
            }
            n = part_sum(n);
            if (i < nblk && part == 0) count[i] = n;
        }
        __syncthreads();
        for (int i0 = 0; i0 < nblk; i0 += ORDER_THREADS / ORDER_PARTS) {
            const int i = i0 + threadIdx.x / ORDER_PARTS;
            int rank = 0;
            if (i < nblk) {
                const int n = count[i];
                for (int j = part; j < nblk; j += ORDER_PARTS) rank += count[j] > n || (count[j] == n && j < i);
            }
            rank = part_sum(rank);
            if (i < nblk && part == 0) {
                (side ? a.order_k : a.order_q)[(long)b * nblk + rank] = i;
                if (alike && a.order_k) a.order_k[(long)b * nblk + rank] = i;
            }
        }
    }
}

// ---- the tiles a row block walks, 64 at a time, one per lane: seen by some row of the workgroup; of those, not by every row in whole; seen by
// the wave; seen by every row of the wave in whole
struct Walk { unsigned long long see, part, wsee, wwhole; };
__device__ __forceinline__ int take_tile(unsigned long long& see) { const int i = __builtin_ctzll(see); see &= see - 1; return i; }

// scores in registers: CAP -> log2 units, otherwise q.k stays as it is (the exponential takes the factor) and the bias comes in q.k's units.
// kslope: slope / scale, or with CAP slope log2(e).  steep: (1 - tanh^2) / 4
// cap tanh(s / cap) as cap - 2 cap u is off by up to cap 2^-21 whatever the score (u, near 1/2, is known to 2^-23): for caps up to CAP_NEAR at most
// 2^-13, a 32nd of what the rounding of p to bf16 may be.  Above it scores below 0.35 cap come from tanh's series and all are within 2^-20 of
// their value.  One kernel with both forms would hold the registers of the larger one and more (dq at head width 64 spills 124 bytes a lane
// instead of 44, at 32 it runs three waves per SIMD instead of four), so each is compiled by itself.  The series costs (caps of 250 and 260, us forward
// and backward): 8 x 12 heads of 1024 tokens in five documents 41 and 45, 110 and 131; 16 over 4 heads of 2048 without masks 79 and 100, 231 and 301.
enum { NEAR = 1, FAR = 2 };                   // the forms of a cap; 0: none
constexpr float CAP_NEAR = 256.f;
template <int CAP, bool BIAS, bool STEEP>
__device__ __forceinline__ void modify(f32x16& s, f32x16& steep, const ModArgs& a, const float (&mine)[3], const float* pos, int row0, float kslope, int lane) {
    if (CAP) {
        const float up = 2.f * a.scale * LOG2E_F / a.cap, capl = a.cap * LOG2E_F;
        if (CAP == NEAR) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float u = __builtin_amdgcn_rcpf(fast_exp2(s[r] * up) + 1.f);                     // tanh(x) = 1 - 2 u, u = 1 / (e^2x + 1)
                s[r] = fmaf(u, -2.f * capl, capl);
                if (STEEP) steep[r] = fmaf(-u, u, u);                                                  // 1 - tanh^2 = 4 (u - u^2)
            }
        } else {
            const float raw = a.scale * LOG2E_F;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float y = s[r] * up, x = y * (0.5f * LN2_F), z = x * x;
                // tanh(x) / x up to x^8; 1382 / 155925 x^10 is left out
                const float t = fmaf(fmaf(fmaf(fmaf(z, 62.f / 2835.f, -17.f / 315.f), z, 2.f / 15.f), z, -1.f / 3.f), z, 1.f);
                const float u = __builtin_amdgcn_rcpf(fast_exp2(y) + 1.f);
                s[r] = fabsf(x) < 0.35f ? s[r] * raw * t : fmaf(u, -2.f * capl, capl);
                if (STEEP) steep[r] = fmaf(-u, u, u);
            }
        }
    }
    if (BIAS) {
        f32x16 far;                                              // signed for one axis: |.| is free where it is used
#pragma unroll
        for (int ax = 0; ax < 3; ++ax) if (ax < a.axes) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 p = *reinterpret_cast<const float4*>(pos + ax * TT + row0 + 8 * g + 4 * (lane >> 5));
                const float d[4] = {p.x - mine[ax], p.y - mine[ax], p.z - mine[ax], p.w - mine[ax]};
#pragma unroll
                for (int e = 0; e < 4; ++e) far[4 * g + e] = ax == 0 ? d[e] : fabsf(far[4 * g + e]) + fabsf(d[e]);
            }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fmaf(fabsf(far[r]), -kslope, s[r]);
    }
}

// What a lane sees of a staged tile, one bit per row.  Documents: for every document among the wave's rows (one or two as a rule) one ballot over the
// tile's rows, `theirs` = the document of the tile's row `lane`.  Order: rows below `left` (BELOW) or from it on.
template <bool BELOW>
__device__ __forceinline__ unsigned long long seen_rows(int left, bool bydoc, int mydoc, int theirs) {
    const unsigned long long upto = left <= 0 ? 0ull : (left >= 64 ? ~0ull : (1ull << left) - 1);
    unsigned long long m = BELOW ? upto : ~upto;
    if (bydoc) {
        unsigned long long same = 0, todo = __builtin_amdgcn_ballot_w64(mydoc >= 0);
        while (todo) {
            const int d = __builtin_amdgcn_readlane(mydoc, __builtin_ctzll(todo));
            const unsigned long long rows = __builtin_amdgcn_ballot_w64(theirs == d);
            if (mydoc == d) same = rows;
            todo &= ~__builtin_amdgcn_ballot_w64(mydoc == d);
        }
        m &= same;
    }
    return m;
}
// does no lane of the wave see any of the 32 rows of half kb (a document that ends in the other half, keys behind the last visible one)
__device__ __forceinline__ bool none_seen(unsigned long long seen, int kb) { return __builtin_amdgcn_ballot_w64((unsigned)(seen >> (kb * 32)) != 0) == 0; }
// accumulator register r of a lane stands for row 8 (r >> 2) + (r & 3) of its block behind the lane's first one; rows that are not seen take `value`
__device__ __forceinline__ void hide(f32x16& x, unsigned long long seen, int kb, int lane, float value) {
    const int bits = (int)((unsigned)(seen >> (kb * 32)) >> (4 * (lane >> 5)));
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        int t;                                                    // all ones or none; as asm, because the compiler turns the builtin into a compare and a select
        asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(t) : "v"(bits), "n"(8 * (r >> 2) + (r & 3)));
        x[r] = __int_as_float((t & __float_as_int(x[r])) | (~t & __float_as_int(value)));
    }
}

// four elements of o, and for the backward pass what their rounding left out
__device__ __forceinline__ void store_o(const ModArgs& a, long at, const float4 v) {
    const uint2 w = make_uint2(pack_bf2(v.x, v.y), pack_bf2(v.z, v.w));
    *reinterpret_cast<uint2*>(a.o + at) = w;
    if (a.o_rest)
        *reinterpret_cast<uint2*>(a.o_rest + at) = make_uint2(pack_bf2(v.x - __uint_as_float(w.x << 16), v.y - __uint_as_float(w.x & 0xffff0000u)),
                                                             pack_bf2(v.z - __uint_as_float(w.y << 16), v.w - __uint_as_float(w.y & 0xffff0000u)));
}

// ================================================ forward ===============================================
// NW waves of 32 queries.  NW = 1 serves up to 32 queries (a pooled or a single new token): every workgroup is one wave, and the keys are
// split over many of them.  NW = 4 otherwise: two waves would stage every tile for half as many queries (a fifth slower on 16 heads of 8192 packed
// tokens).  Three waves per SIMD (16 heads of 4095 tokens behind a prefix: 100 us in three and in two, 107 in four); with a distance bias the
// registers are those of two (64 x 12 heads of 257 tokens with lse: 61 us, 64 when held to three; 16 heads of 8192 packed tokens 73 and 72).
template <int HD, int NW, int CAP, bool BIAS>
__global__ __launch_bounds__(64 * NW, BIAS ? 2 : 3) void attn_mod_fwd_kernel(const ModArgs a) {
    constexpr int KS = HD / 16, DJ = HD / 32, NT = 64 * NW, TB = TT * HD * 2;
    __shared__ __attribute__((aligned(16))) char ldsK[2][TB];
    __shared__ __attribute__((aligned(16))) char ldsV[2][TB];
    __shared__ __attribute__((aligned(16))) float ldsP[2][BIAS ? 3 * TT : 4];
    __shared__ unsigned long long noted[3];                      // of tile n: slot n % 3
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int bh, blk;
    place(blockIdx.x, a.B * a.H, a.nblk * a.splits, a.abreast, bh, blk);
    const int split = blk % a.splits, b = bh / a.H, h = bh - b * a.H, hk = h / a.G;
    blk /= a.splits;
    if (a.order) blk = a.order[(long)b * a.nblk + blk];
    else if (a.causal) blk = a.nblk - 1 - blk;                  // the last queries see the most
    const bf16_t* kp = a.k + (long)b * a.k_bs + (long)hk * a.k_hs;
    const bf16_t* vp = a.v + (long)b * a.v_bs + (long)hk * a.v_hs;
    const int* docs = a.doc_k ? a.doc_k + (long)b * a.Nk : nullptr;
    const int4* tab = a.tab_k ? a.tab_k + (long)b * a.ntk : nullptr;
    const float* posk = BIAS ? a.pos_k + (long)b * a.Nk * a.axes : nullptr;
    const int off = a.Nk - a.Nq;
    const int pre = a.causal ? (a.prefix ? min(max(a.prefix[b], 0), a.Nk) : 0) : a.Nk;
    // this lane's query (rows behind the last one repeat it and are not stored)
    const int q0 = blk * 32 * NW + wave * 32, qr = min(q0 + (lane & 31), a.Nq - 1);
    const bool active = q0 < a.Nq;
    const bf16_t* qp = a.q + (long)b * a.q_bs + (long)qr * a.q_rs + (long)h * a.q_hs;
    bf16x8 qf[KS];
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) qf[kk] = *reinterpret_cast<const bf16x8*>(qp + kk * 16 + 8 * (lane >> 5));
    float mine[3] = {0.f, 0.f, 0.f};
    float kslope = 0.f;
    if (BIAS) {
        kslope = CAP ? a.slopes[h] * LOG2E_F : a.slopes[h] / a.scale;
        for (int ax = 0; ax < a.axes; ++ax) mine[ax] = a.pos_q[((long)b * a.Nq + qr) * a.axes + ax];
    }
    auto lim_of = [&](int i) { return max(pre, min(i + off + 1, a.Nk)); };               // keys below it are visible as far as order goes (may be <= 0)
    const int mydoc = a.doc_q ? a.doc_q[(long)b * a.Nq + qr] : 0;
    const int lim = mydoc < 0 ? 0 : lim_of(qr);                  // padding sees nothing
    const int wlim_lo = lim_of(min(q0, a.Nq - 1)), wlim_hi = lim_of(min(q0 + 31, a.Nq - 1));      // (documents are tested apart)
    int wlo = 0, whi = 0;
    bool pure = true;
    if (tab) {
        wlo = __builtin_amdgcn_readfirstlane(wave_min_i(mydoc < 0 ? 0x7fffffff : mydoc));
        whi = __builtin_amdgcn_readfirstlane(wave_max_i(mydoc));
        pure = wlo == whi && __builtin_amdgcn_ballot_w64(mydoc < 0) == 0;
    }
    // the workgroup's ranges: over its 64-row document tiles, and by its first and last row
    const int g0 = blk * 32 * NW, g1 = min(g0 + 32 * NW, a.Nq) - 1;
    const int glim_lo = lim_of(g0), glim_hi = lim_of(g1);
    int glo = 0, ghi = 0;
    bool gpure = true;
    if (tab) {
        glo = 0x7fffffff; ghi = -1;
        for (int t = g0 / TT; t <= g1 / TT; ++t) {
            const int4 e = a.tab_q[(long)b * a.ntq + t];
            glo = min(glo, e.x); ghi = max(ghi, e.y);
            gpure &= e.z == min(TT, a.Nq - t * TT);
        }
        gpure &= glo == ghi;
    }
    f32x16 o[DJ];
#pragma unroll
    for (int dj = 0; dj < DJ; ++dj) o[dj] = zero16();
    float m_run = -INFINITY, l_run = 0.f;
    bool poisoned = false;
    constexpr bool RAW = !CAP;                                   // scores stay in q.k's units and the exponential takes the factor
    const float unit = RAW ? a.scale * LOG2E_F : 1.f;

    RowFrag<HD> fk; fk.init(lane);
    ColFrag<HD> fv; fv.init(lane);
    Dma<HD, NW> dk, dv;
    dk.init(a.k_rs, lane, wave); dv.init(a.v_rs, lane, wave);
    constexpr int AXW = (3 + NW - 1) / NW;                       // the waves share the axes
    float pv[AXW] = {}; int dc = 0, dn = 0;                      // documents of the tile's rows, one per lane: of this tile and of the next
    auto fetch = [&](int t, int buf) {
        dk.fetch(kp, t * TT, a.Nk, ldsK[buf], lane, wave);
        dv.fetch(vp, t * TT, a.Nk, ldsV[buf], lane, wave);
        const int r = min(t * TT + lane, a.Nk - 1);
        if (BIAS) {
#pragma unroll
            for (int x = 0; x < AXW; ++x) if (wave + NW * x < a.axes) pv[x] = posk[(long)r * a.axes + wave + NW * x];
        }
        if (docs) dn = docs[r];
    };
    auto land = [&](int buf, int slot, bool partial) {
        if (BIAS) {
#pragma unroll
            for (int x = 0; x < AXW; ++x) if (wave + NW * x < a.axes) ldsP[buf][(wave + NW * x) * TT + lane] = pv[x];
        }
        dc = dn;
        dma_landed();
        if (partial) dv.tidy(ldsV[buf], &noted[slot], lane, wave);
    };
    if (tid < 3) noted[tid] = 0;
    __syncthreads();
    int buf = 0, slot = 0;
    // a split walks every splits-th tile (runs of neighbouring tiles would be unequal under an order or documents)
    const int nmine = (a.ntk - split + a.splits - 1) / a.splits;
    for (int base = 0; base < nmine; base += 64) {
    Walk wk;
    {
        const int i = base + lane, t = split + i * a.splits;
        bool see = i < nmine && t * TT < glim_hi, whole = t * TT + TT <= glim_lo;
        bool ws = see && active && t * TT < wlim_hi, ww = t * TT + TT <= wlim_lo;
        if (docs && !tab) whole = ww = false;
        if (tab && see) {
            const int4 e = tab[t];
            see = e.x <= ghi && e.y >= glo;
            whole = whole && gpure && e.x == e.y && e.x == glo && e.z == TT;
            ws = ws && e.x <= whi && e.y >= wlo;
            ww = ww && pure && e.x == e.y && e.x == wlo && e.z == TT;
        }
        wk.see = __builtin_amdgcn_ballot_w64(see);
        wk.part = __builtin_amdgcn_ballot_w64(see && !whole);
        wk.wsee = __builtin_amdgcn_ballot_w64(ws);
        wk.wwhole = __builtin_amdgcn_ballot_w64(ww);
    }
    if (wk.see == 0) continue;
    int i = take_tile(wk.see);
    fetch(split + (base + i) * a.splits, buf);
    land(buf, slot, (wk.part >> i) & 1);
    __syncthreads();
    while (true) {
        const int in = wk.see ? take_tile(wk.see) : -1;
        if (in >= 0) fetch(split + (base + in) * a.splits, buf ^ 1);
        const int slot_n = slot == 2 ? 0 : slot + 1;
        if (tid == 0) noted[slot_n == 2 ? 0 : slot_n + 1] = 0;   // read during the tile before this one, written during the next one
        const int j0 = (split + (base + i) * a.splits) * TT;
        const bool see = (wk.wsee >> i) & 1, whole = (wk.wwhole >> i) & 1;
        if (see) {
            unsigned long long seen = ~0ull;
            if (!whole) seen = seen_rows<true>(lim - j0, docs != nullptr, mydoc, dc);
            const uint32_t kt = lds_addr(ldsK[buf]), vt = lds_addr(ldsV[buf]);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                if (!whole && none_seen(seen, kb)) continue;
                f32x16 s = zero16();
#pragma unroll
                for (int kk = 0; kk < KS; ++kk) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fk.read(kt, kb * 32, kk), qf[kk], s, 0, 0, 0);
                modify<CAP, BIAS, false>(s, s, a, mine, ldsP[buf], kb * 32, kslope, lane);
                if (!whole) hide(s, seen, kb, lane, -INFINITY);
                float mx = s[0];
#pragma unroll
                for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
                const float2 mh = halves(mx);
                // the reference point moves only when some row of the wave outgrew it by 2^8 (p <= 256 instead of 1): most blocks then skip
                // the rescale of the 16 HD / 32 output registers
                const float m_new = fmaxf(m_run, fmaxf(mh.x, mh.y));
                if (__builtin_amdgcn_ballot_w64((m_new - m_run) * unit > 8.f)) {
                    const float alpha = m_run == -INFINITY ? 0.f : fast_exp2((m_run - m_new) * unit);
                    m_run = m_new;
                    l_run *= alpha;
#pragma unroll
                    for (int dj = 0; dj < DJ; ++dj)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[dj][r] *= alpha;
                }
                const float mu = m_run == -INFINITY ? 0.f : m_run * unit;
                float l0 = 0.f, l1 = 0.f;
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    s[r] = fast_exp2(RAW ? fmaf(s[r], unit, -mu) : s[r] - mu);
                    s[r + 1] = fast_exp2(RAW ? fmaf(s[r + 1], unit, -mu) : s[r + 1] - mu);
                    l0 += s[r]; l1 += s[r + 1];
                }
                l_run += l0 + l1;
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const bf16x8 p = pack_half(s, m);
#pragma unroll
                    for (int dj = 0; dj < DJ; ++dj) o[dj] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fv.read(vt, kb * 32 + 16 * m, dj), p, o[dj], 0, 0, 0);
                }
            }
            if (((wk.part >> i) & 1) && (noted[slot] & seen)) poisoned = true;
        }
        if (in >= 0) land(buf ^ 1, slot_n, (wk.part >> in) & 1);
        __syncthreads();
        buf ^= 1; slot = slot_n;
        if (in < 0) break;
        i = in;
    }
    }
    const float2 lh = halves(l_run);
    l_run = lh.x + lh.y;
    if (poisoned) l_run = NAN;
    const int row = q0 + (lane & 31);
    if (row >= a.Nq) return;
    if (a.splits > 1) {
        const long rows = (long)a.B * a.H * a.Nq, at = ((long)split * rows + ((long)b * a.H + h) * a.Nq + row);
#pragma unroll
        for (int dj = 0; dj < DJ; ++dj)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<float4*>(a.part + at * HD + dj * 32 + 8 * g + 4 * (lane >> 5)) = make_float4(o[dj][4 * g], o[dj][4 * g + 1], o[dj][4 * g + 2], o[dj][4 * g + 3]);
        if (lane < 32) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m_run * unit, l_run);
        return;
    }
    const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
    const long at = (long)b * a.o_bs + (long)row * a.o_rs + (long)h * a.o_hs;
#pragma unroll
    for (int dj = 0; dj < DJ; ++dj)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            store_o(a, at + dj * 32 + 8 * g + 4 * (lane >> 5), make_float4(o[dj][4 * g] * inv, o[dj][4 * g + 1] * inv, o[dj][4 * g + 2] * inv, o[dj][4 * g + 3] * inv));
    if (a.lse && lane < 32) a.lse[((long)b * a.H + h) * a.Nq + row] = l_run == 0.f ? -INFINITY : (m_run * unit + __log2f(l_run)) * LN2_F;
}

// joins the splits of a row: weights 2^(m_s - max m).  A wave per row: 4 elements a lane, the splits dealt over the 256 / HD groups of lanes (one
// thread per 4 elements walked its splits one load after the other: 10 us for 192 rows of 11)
template <int HD>
__global__ __launch_bounds__(256) void attn_mod_join_kernel(const ModArgs a) {
    constexpr int CPR = HD / 4, NG = 64 / CPR;
    const long rows = (long)a.B * a.H * a.Nq, r = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= rows) return;
    const int lane = threadIdx.x & 63, c = (lane % CPR) * 4, g = lane / CPR;
    float m = lane < a.splits ? a.part_ml[(lane * rows + r) * 2] : -INFINITY;      // at most 64 splits
    m = wave_max(m);
    float l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = g; s < a.splits; s += NG) {
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + (s * rows + r) * 2);
        const float4 v = *reinterpret_cast<const float4*>(a.part + (s * rows + r) * HD + c);
        // a split that saw nothing has m = -inf, l = 0 and o = 0; a row that is NaN without a maximum stays NaN
        const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : fast_exp2(ml.x - m);
        l = fmaf(ml.y, f, l);
        acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
    }
#pragma unroll
    for (int o = CPR; o < 64; o <<= 1) {
        l += __shfl_xor(l, o, 64);
        acc.x += __shfl_xor(acc.x, o, 64); acc.y += __shfl_xor(acc.y, o, 64); acc.z += __shfl_xor(acc.z, o, 64); acc.w += __shfl_xor(acc.w, o, 64);
    }
    if (g != 0) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const long bh = r / a.Nq;
    const int row = (int)(r - bh * a.Nq), b = (int)(bh / a.H), h = (int)(bh - (long)b * a.H);
    store_o(a, (long)b * a.o_bs + (long)row * a.o_rs + (long)h * a.o_hs + c, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    if (a.lse && c == 0) a.lse[r] = l == 0.f ? -INFINITY : (m + __log2f(l)) * LN2_F;
}

// ================================================ backward ==============================================
// The two owner kernels share the walk, the staging and the arithmetic of a 32 x 32 block:
//   OWN_Q: lane = query, tiles of keys:  S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T          (8 hd flop a pair, ds in two parts)
//   OWN_K: lane = key, tiles of queries: S = Q K^T,  dP = dO V^T,  dV^T += dO^T P, dK^T += Q^T dS         (10 hd)
// Scores and dP are formed twice (4 hd of the 18), which costs less than the atomics or the traffic of dq partials that one kernel would need: a
// tile of 64 keys would add 64 KiB of fp32 to HBM for every 128 queries.  Four waves of 32 rows; dq runs at three waves per SIMD
// (the pass above 375 us, 378 in two; 8 x 12 heads of 1024 in five documents, capped, 110 and 115), dk / dv and a distance bias at two: in three they
// spill (375 -> 509 us; 16 heads of 8192 packed tokens with a distance 200 -> 295).
// X, Y: the staged matrices (K, V or Q, dO); own fragments: (Q, dO) or (K, V).  OWN_Q also forms sum(do o), which OWN_K reads.
template <int HD, bool OWN_Q, int CAP, bool BIAS>
__global__ __launch_bounds__(256, OWN_Q && !BIAS ? 3 : 2) void attn_mod_bwd_kernel(const ModArgs a) {
    constexpr int KS = HD / 16, DJ = HD / 32, TB = TT * HD * 2;
    __shared__ __attribute__((aligned(16))) char ldsX[2][TB];
    __shared__ __attribute__((aligned(16))) char ldsY[2][TB];
    __shared__ __attribute__((aligned(16))) float ldsP[2][BIAS ? 3 * TT : 4];
    __shared__ __attribute__((aligned(16))) float ldsL[2][OWN_Q ? 4 : 2 * TT];      // lse (log2 units) and sum(do o) of the staged queries
    __shared__ unsigned long long noted[3];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int OH = OWN_Q ? a.H : a.Hk;                                               // the owner's head: a query head or a key head
    int bo, blk;
    const unsigned id = blockIdx.y * gridDim.x + blockIdx.x;                         // (a second dimension from 2^24 workgroups on)
    if (id >= (unsigned)(a.B * OH) * a.nblk * a.splits) return;
    place((int)id, a.B * OH, a.nblk * a.splits, a.abreast, bo, blk);
    const int split = blk % a.splits, b = bo / OH, ho = bo - b * OH;
    blk /= a.splits;
    if (a.order) blk = a.order[(long)b * a.nblk + blk];
    else if (OWN_Q && a.causal) blk = a.nblk - 1 - blk;                                   // the last queries see the most, the first keys are seen the most
    const int NO = OWN_Q ? a.Nq : a.Nk, NS = OWN_Q ? a.Nk : a.Nq;                    // rows of the owner's side and of the staged side
    const int off = a.Nk - a.Nq;
    const int pre = a.causal ? (a.prefix ? min(max(a.prefix[b], 0), a.Nk) : 0) : a.Nk;
    const bool bydoc = a.doc_k != nullptr;
    const int* doc_o = bydoc ? (OWN_Q ? a.doc_q : a.doc_k) + (long)b * NO : nullptr;
    const int* doc_s = bydoc ? (OWN_Q ? a.doc_k : a.doc_q) + (long)b * NS : nullptr;
    const int nts = OWN_Q ? a.ntk : a.ntq, nto = OWN_Q ? a.ntq : a.ntk;
    const int4* tab_s = a.tab_k ? (OWN_Q ? a.tab_k : a.tab_q) + (long)b * nts : nullptr;
    const int4* tab_o = a.tab_k ? (OWN_Q ? a.tab_q : a.tab_k) + (long)b * nto : nullptr;
    const float* pos_s = BIAS ? (OWN_Q ? a.pos_k : a.pos_q) + (long)b * NS * a.axes : nullptr;
    const int r0 = blk * 128 + wave * 32, ro = min(r0 + (lane & 31), NO - 1), row = r0 + (lane & 31);
    const bool active = r0 < NO;
    // own fragments
    bf16x8 fa[KS], fb[KS];
    float lse2 = 0.f, D = 0.f;
    {
        const bf16_t* pa = OWN_Q ? a.q + (long)b * a.q_bs + (long)ro * a.q_rs + (long)ho * a.q_hs : a.k + (long)b * a.k_bs + (long)ro * a.k_rs + (long)ho * a.k_hs;
        const bf16_t* pb = OWN_Q ? a.d_o + (long)b * a.do_bs + (long)ro * a.do_rs + (long)ho * a.do_hs : a.v + (long)b * a.v_bs + (long)ro * a.v_rs + (long)ho * a.v_hs;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
            fa[kk] = *reinterpret_cast<const bf16x8*>(pa + kk * 16 + 8 * (lane >> 5));
            fb[kk] = *reinterpret_cast<const bf16x8*>(pb + kk * 16 + 8 * (lane >> 5));
        }
        if (OWN_Q) {
            const long at_o = (long)b * a.o_bs + (long)ro * a.o_rs + (long)ho * a.o_hs;
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                const bf16x8 fo = *reinterpret_cast<const bf16x8*>(a.o + at_o + kk * 16 + 8 * (lane >> 5));
                bf16x8 rest = {0, 0, 0, 0, 0, 0, 0, 0};
                if (a.o_rest) rest = *reinterpret_cast<const bf16x8*>(a.o_rest + at_o + kk * 16 + 8 * (lane >> 5));
#pragma unroll
                for (int e = 0; e < 8; ++e) D = fmaf(bf2f((bf16_t)fo[e]) + bf2f((bf16_t)rest[e]), bf2f((bf16_t)fb[kk][e]), D);
            }
            const float2 dh = halves(D);
            D = dh.x + dh.y;
            const long at = ((long)b * a.H + ho) * a.Nq + ro;
            lse2 = a.lse[at] * LOG2E_F;
            if (lse2 == -INFINITY) { lse2 = INFINITY; D = 0.f; }                     // a row that saw nothing: p = 2^(s - inf) = 0
            if (split == 0 && lane < 32 && row < NO) a.dsum[at] = D;
        }
    }
    const int mydoc = bydoc ? doc_o[ro] : 0;
    float mine[3] = {0.f, 0.f, 0.f};
    if (BIAS) for (int ax = 0; ax < a.axes; ++ax) mine[ax] = (OWN_Q ? a.pos_q : a.pos_k)[((long)b * NO + ro) * a.axes + ax];
    // order: the staged index must be below `edge` (OWN_Q) or at least `edge` (OWN_K); first and last row of the wave and of the workgroup
    auto edge_of = [&](int r) { return OWN_Q ? max(pre, min(r + off + 1, a.Nk)) : (r < pre ? 0 : r - off); };
    const int edge = mydoc >= 0 ? edge_of(ro) : (OWN_Q ? 0 : 1 << 30);                // padding sees nothing and is seen by nothing
    const int w1 = min(r0 + 32, NO) - 1, g0 = blk * 128, g1 = min(g0 + 128, NO) - 1;
    const int wedge0 = edge_of(min(r0, NO - 1)), wedge1 = edge_of(w1), gedge0 = edge_of(g0), gedge1 = edge_of(g1);
    int wlo = 0, whi = 0, glo = 0, ghi = 0;
    bool pure = true, gpure = true;
    if (tab_s) {
        wlo = __builtin_amdgcn_readfirstlane(wave_min_i(mydoc < 0 ? 0x7fffffff : mydoc));
        whi = __builtin_amdgcn_readfirstlane(wave_max_i(mydoc));
        pure = wlo == whi && __builtin_amdgcn_ballot_w64(mydoc < 0) == 0;
        glo = 0x7fffffff; ghi = -1;
        for (int t = g0 / TT; t <= g1 / TT; ++t) {
            const int4 e = tab_o[t];
            glo = min(glo, e.x); ghi = max(ghi, e.y);
            gpure &= e.z == min(TT, NO - t * TT);
        }
        gpure &= glo == ghi;
    }
    auto order_see = [&](int t, int e0, int e1) { return OWN_Q ? t * TT < e1 : t * TT + TT > e0; };
    auto order_whole = [&](int t, int e0, int e1) { return OWN_Q ? t * TT + TT <= e0 : t * TT >= e1; };
    f32x16 ga[DJ], gb[OWN_Q ? 1 : DJ];                           // dQ^T, or dK^T and dV^T
#pragma unroll
    for (int dj = 0; dj < DJ; ++dj) { ga[dj] = zero16(); if (!OWN_Q) gb[dj] = zero16(); }
    bool poisoned = false;
    constexpr bool RAW = !CAP;
    const float unit = RAW ? a.scale * LOG2E_F : 1.f;

    RowFrag<HD> fr; fr.init(lane);
    ColFrag<HD> fc; fc.init(lane);
    Dma<HD, 4> dx, dy;
    dx.init(OWN_Q ? a.k_rs : a.q_rs, lane, wave); dy.init(OWN_Q ? a.v_rs : a.do_rs, lane, wave);
    float pv = 0.f, lv = 0.f; int dc = 0, dn = 0;
    const bf16_t *X = nullptr, *Y = nullptr;
    const float* rowv = nullptr;                                 // OWN_K: wave 0 reads lse, wave 1 sum(do o)
    auto fetch = [&](int t, int buf) {
        dx.fetch(X, t * TT, NS, ldsX[buf], lane, wave);
        dy.fetch(Y, t * TT, NS, ldsY[buf], lane, wave);
        const int r = min(t * TT + lane, NS - 1);
        if (BIAS && wave < a.axes) pv = pos_s[(long)r * a.axes + wave];
        if (bydoc) dn = doc_s[r];
        if (!OWN_Q && wave < 2) lv = rowv[r];
    };
    auto land = [&](int t, int buf, int slot, bool partial) {
        if (BIAS && wave < a.axes) ldsP[buf][wave * TT + lane] = pv;
        dc = dn;
        if (!OWN_Q && wave < 2) {
            // negated: raw scores and dp start from them in the accumulators; behind the last query and in rows that saw nothing p = 0
            const bool in = t * TT + lane < NS;
            if (wave == 0) ldsL[buf][lane] = (in && lv != -INFINITY) ? lv * (-LOG2E_F / unit) : -INFINITY;
            else ldsL[buf][TT + lane] = in ? -lv : 0.f;
        }
        dma_landed();
        if (partial) {
            dx.tidy(ldsX[buf], &noted[slot], lane, wave);
            if (!OWN_Q) dy.tidy(ldsY[buf], &noted[slot], lane, wave);
        }
    };
    if (tid < 3) noted[tid] = 0;
    __syncthreads();
    int buf = 0, slot = 0;
    const int nmine = (nts - split + a.splits - 1) / a.splits;   // a split walks every splits-th tile
    for (int g = 0; g < (OWN_Q ? 1 : a.G); ++g) {
    const int h = OWN_Q ? ho : ho * a.G + g;
    X = OWN_Q ? a.k + (long)b * a.k_bs + (long)(ho / a.G) * a.k_hs : a.q + (long)b * a.q_bs + (long)h * a.q_hs;
    Y = OWN_Q ? a.v + (long)b * a.v_bs + (long)(ho / a.G) * a.v_hs : a.d_o + (long)b * a.do_bs + (long)h * a.do_hs;
    if (!OWN_Q) rowv = (wave ? a.dsum : a.lse) + ((long)b * a.H + h) * a.Nq;
    for (int base = 0; base < nmine; base += 64) {
    Walk wk;
    {
        const int i = base + lane, t = split + i * a.splits;
        bool see = i < nmine && order_see(t, gedge0, gedge1), whole = order_whole(t, gedge0, gedge1) && t * TT + TT <= NS;
        bool ws = see && active && order_see(t, wedge0, wedge1), ww = order_whole(t, wedge0, wedge1) && (!OWN_Q || t * TT + TT <= NS);
        if (bydoc && !tab_s) whole = ww = false;
        if (tab_s && see) {
            const int4 e = tab_s[t];
            see = e.x <= ghi && e.y >= glo;
            whole = whole && gpure && e.x == e.y && e.x == glo && e.z == TT;
            ws = ws && e.x <= whi && e.y >= wlo;
            ww = ww && pure && e.x == e.y && e.x == wlo && e.z == TT;
        }
        wk.see = __builtin_amdgcn_ballot_w64(see);
        wk.part = __builtin_amdgcn_ballot_w64(see && !whole);
        wk.wsee = __builtin_amdgcn_ballot_w64(ws);
        wk.wwhole = __builtin_amdgcn_ballot_w64(ww);
    }
    if (wk.see == 0) continue;
    int i = take_tile(wk.see);
    { const int t = split + (base + i) * a.splits; fetch(t, buf); land(t, buf, slot, (wk.part >> i) & 1); }
    __syncthreads();
    while (true) {
        const int in = wk.see ? take_tile(wk.see) : -1, tn = split + (base + in) * a.splits;
        if (in >= 0) fetch(tn, buf ^ 1);
        const int slot_n = slot == 2 ? 0 : slot + 1;
        if (tid == 0) noted[slot_n == 2 ? 0 : slot_n + 1] = 0;   // read during the tile before this one, written during the next one
        const int j0 = (split + (base + i) * a.splits) * TT;
        const bool see = (wk.wsee >> i) & 1, whole = (wk.wwhole >> i) & 1;
        if (see) {
            unsigned long long seen = ~0ull;
            if (!whole) seen = seen_rows<OWN_Q>(edge - j0, bydoc, mydoc, dc);
            const float kslope = !BIAS ? 0.f : (CAP ? a.slopes[h] * LOG2E_F : a.slopes[h] / a.scale);
            const uint32_t xb = lds_addr(ldsX[buf]), yb = lds_addr(ldsY[buf]);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                if (OWN_Q ? j0 + kb * 32 >= wedge1 : j0 + kb * 32 >= NS) break;
                if (!OWN_Q && j0 + kb * 32 + 32 <= wedge0) continue;
                f32x16 s = zero16(), dp = zero16(), steep;
                if (!OWN_Q) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int jr = kb * 32 + 8 * q + 4 * (lane >> 5);
                        if (RAW) { const float4 L = *reinterpret_cast<const float4*>(&ldsL[buf][jr]); s[4 * q] = L.x; s[4 * q + 1] = L.y; s[4 * q + 2] = L.z; s[4 * q + 3] = L.w; }
                        const float4 E = *reinterpret_cast<const float4*>(&ldsL[buf][TT + jr]);
                        dp[4 * q] = E.x; dp[4 * q + 1] = E.y; dp[4 * q + 2] = E.z; dp[4 * q + 3] = E.w;
                    }
                }
#pragma unroll
                for (int kk = 0; kk < KS; ++kk) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr.read(xb, kb * 32, kk), fa[kk], s, 0, 0, 0);
#pragma unroll
                for (int kk = 0; kk < KS; ++kk) dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr.read(yb, kb * 32, kk), fb[kk], dp, 0, 0, 0);
                modify<CAP, BIAS, true>(s, steep, a, mine, ldsP[buf], kb * 32, kslope, lane);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float4 L = make_float4(-lse2, -lse2, -lse2, -lse2);
                    if (!OWN_Q && !RAW) L = *reinterpret_cast<const float4*>(&ldsL[buf][kb * 32 + 8 * q + 4 * (lane >> 5)]);
                    const float Ls[4] = {L.x, L.y, L.z, L.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 4 * q + e;
                        s[r] = fast_exp2(!RAW ? s[r] + Ls[e] : (OWN_Q ? fmaf(s[r], unit, Ls[e]) : s[r] * unit));
                        dp[r] = OWN_Q ? s[r] * (dp[r] - D) : s[r] * dp[r];
                        if (CAP) dp[r] *= steep[r];
                    }
                }
                if (!whole) {
                    if (!OWN_Q) hide(s, seen, kb, lane, 0.f);
                    hide(dp, seen, kb, lane, 0.f);
                }
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const bf16x8 ds = pack_half(dp, m), rest = pack_rest(dp, m, ds);
#pragma unroll
                    for (int dj = 0; dj < DJ; ++dj) {
                        const bf16x8 x = fc.read(xb, kb * 32 + 16 * m, dj);
                        ga[dj] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, ds, ga[dj], 0, 0, 0);
                        ga[dj] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, rest, ga[dj], 0, 0, 0);
                    }
                    if (!OWN_Q) {
                        const bf16x8 p = pack_half(s, m);
#pragma unroll
                        for (int dj = 0; dj < DJ; ++dj) gb[dj] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fc.read(yb, kb * 32 + 16 * m, dj), p, gb[dj], 0, 0, 0);
                    }
                }
            }
            if (((wk.part >> i) & 1) && (noted[slot] & seen)) poisoned = true;
        }
        if (in >= 0) land(tn, buf ^ 1, slot_n, (wk.part >> in) & 1);
        __syncthreads();
        buf ^= 1; slot = slot_n;
        if (in < 0) break;
        i = in;
    }
    }
    }
    if (row >= NO) return;
    const float fa_out = poisoned ? NAN : (CAP ? 4.f * a.scale : a.scale), fb_out = poisoned ? NAN : 1.f;
    if (a.splits > 1) {
        const long rows = (long)a.B * OH * NO;
        float* base = a.part + (((long)split * rows + ((long)b * OH + ho) * NO + row) * (OWN_Q ? 1 : 2)) * HD;
#pragma unroll
        for (int dj = 0; dj < DJ; ++dj)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int d = dj * 32 + 8 * q + 4 * (lane >> 5);
                *reinterpret_cast<float4*>(base + d) = make_float4(ga[dj][4 * q] * fa_out, ga[dj][4 * q + 1] * fa_out, ga[dj][4 * q + 2] * fa_out, ga[dj][4 * q + 3] * fa_out);
                if (!OWN_Q) *reinterpret_cast<float4*>(base + HD + d) = make_float4(gb[dj][4 * q] * fb_out, gb[dj][4 * q + 1] * fb_out, gb[dj][4 * q + 2] * fb_out, gb[dj][4 * q + 3] * fb_out);
            }
        return;
    }
    bf16_t* pa = OWN_Q ? a.dq + (long)b * a.dq_bs + (long)row * a.dq_rs + (long)ho * a.dq_hs : a.dk + (long)b * a.dk_bs + (long)row * a.dk_rs + (long)ho * a.dk_hs;
    bf16_t* pb = OWN_Q ? nullptr : a.dv + (long)b * a.dv_bs + (long)row * a.dv_rs + (long)ho * a.dv_hs;
#pragma unroll
    for (int dj = 0; dj < DJ; ++dj)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int d = dj * 32 + 8 * q + 4 * (lane >> 5);
            *reinterpret_cast<uint2*>(pa + d) = make_uint2(pack_bf2(ga[dj][4 * q] * fa_out, ga[dj][4 * q + 1] * fa_out), pack_bf2(ga[dj][4 * q + 2] * fa_out, ga[dj][4 * q + 3] * fa_out));
            if (!OWN_Q) *reinterpret_cast<uint2*>(pb + d) = make_uint2(pack_bf2(gb[dj][4 * q] * fb_out, gb[dj][4 * q + 1] * fb_out), pack_bf2(gb[dj][4 * q + 2] * fb_out, gb[dj][4 * q + 3] * fb_out));
        }
}

// adds the splits of gradient rows in order: [split][rows][sides][HD] fp32 -> bf16, one thread per 4 elements
struct JoinOut { bf16_t* p; long bs, rs, hs; };
__global__ __launch_bounds__(256) void attn_mod_sum_kernel(const float* __restrict__ part, int splits, long rows, int sides, int HD, int OH, int NO, JoinOut o0, JoinOut o1) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    const int per = sides * HD / 4;
    const long r = i / per;
    if (r >= rows) return;
    const int e = (int)(i - r * per) * 4, side = e / HD, c = e - side * HD;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < splits; ++s) {
        const float4 v = *reinterpret_cast<const float4*>(part + (s * rows + r) * sides * HD + e);
        acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
    }
    const long bh = r / NO;
    const int row = (int)(r - bh * NO), b = (int)(bh / OH), h = (int)(bh - (long)b * OH);
    const JoinOut& o = side ? o1 : o0;
    *reinterpret_cast<uint2*>(o.p + (long)b * o.bs + (long)row * o.rs + (long)h * o.hs + c) = make_uint2(pack_bf2(acc.x, acc.y), pack_bf2(acc.z, acc.w));
}

// ================================================ host ==================================================
struct Plan {
    int ntq, ntk, nw, nblk, splits, dq_splits, dkv_splits;
    bool tables, ordered;
    long tab_q, tab_k, order_q, order_k, dsum, part, part_ml, bytes;             // byte offsets into the workspace
};

// Splits of a row's tiles, so that `want` workgroups run.  Partial results are written and read in fp32, so a split keeps the more tiles the better
// the blocks fill the chip by themselves: 4, from 128 blocks on 8, from 256 on 16.  Measured at 8 x 12 heads of 512 tokens (384 blocks of 8
// tiles): 24 us whole, 41 in two splits; 3 x 12 heads of 538 (180 of 9): 22 and 28; causal, 8 heads of 4096 (256 of 64): 83 and 61.  Blocks of
// one wave cost less to join and fill less: half of that, at half as many (one query, us with 2 / 4 / 8 tiles: 32 blocks of 11 tiles 12.0 /
// 16.1 / 21.3, 96 of 24 18.3 / 15.8 / 20.5, 384 of 16 28.1 / 26.1 / 23.2); more than 32 splits only with 8 tiles each (256 tiles, 24 blocks:
// 23.6 us in 32 splits, 27.4 in 64).
int splits_for(long blocks, int waves, long want, int tiles) {
    if (blocks <= 0 || blocks >= want) return 1;
    const int half = waves == 1 ? 2 : 1, least = (blocks * half < 128 ? 4 : (blocks * half < 256 ? 8 : 16)) / half;
    int s = (int)((want + blocks - 1) / blocks);
    if (s > tiles / least) s = tiles / least;
    if (s > 32 && s > tiles / 8) s = tiles / 8 > 32 ? tiles / 8 : 32;
    if (s > MAX_SPLITS) s = MAX_SPLITS;
    return s < 1 ? 1 : s;
}

Plan plan_for(const mrg_attn_mod_desc* d, bool backward) {
    Plan p = {};
    p.ntq = (d->Nq + TT - 1) / TT; p.ntk = (d->Nk + TT - 1) / TT;
    long at = 0;
    auto take = [&](long bytes) { const long o = at; at += (bytes + 255) / 256 * 256; return o; };
    const long rows_q = (long)d->B * d->H * d->Nq, rows_k = (long)d->B * d->Hk * d->Nk;
    if (!backward) {
        // up to 32 queries: workgroups of one wave, four resident per CU, and the keys cut until every CU has its four
        p.nw = d->Nq <= 32 ? 1 : 4;
        p.nblk = (d->Nq + 32 * p.nw - 1) / (32 * p.nw);
        p.splits = splits_for((long)d->B * d->H * p.nblk, p.nw, p.nw == 1 ? 2048 : 512, p.ntk);
        p.tables = d->doc_k && (p.nw == 1 ? p.ntk > 2 : p.ntk > 4);
        if (p.splits > 1) { p.part = take(4l * p.splits * rows_q * d->head_dim); p.part_ml = take(8l * p.splits * rows_q); }
    } else {
        p.dsum = take(4l * rows_q);
        p.tables = d->doc_k && (p.ntk > 4 || p.ntq > 4);
        p.dq_splits = splits_for((long)d->B * d->H * ((d->Nq + 127) / 128), 4, 512, p.ntk);
        p.dkv_splits = splits_for((long)d->B * d->Hk * ((d->Nk + 127) / 128), 4, d->causal ? 1024 : 512, p.ntq * (d->H / d->Hk));
        if (p.dkv_splits > p.ntq) p.dkv_splits = p.ntq ? p.ntq : 1;
        long part = 0;
        if (p.dq_splits > 1) part = 4l * p.dq_splits * rows_q * d->head_dim;
        if (p.dkv_splits > 1 && 8l * p.dkv_splits * rows_k * d->head_dim > part) part = 8l * p.dkv_splits * rows_k * d->head_dim;
        p.part = take(part);                                    // used by dq first, by dk / dv behind it
    }
    if (p.tables) {
        p.tab_q = take(16l * d->B * p.ntq); p.tab_k = take(16l * d->B * p.ntk);
        // more than two workgroups per CU, and tables that one workgroup per batch row makes in a few microseconds (2 - 3 us more than the tables
        // alone: 8 x 12 heads of 1024 tokens, 768 blocks, 49 -> 42 us forward; 6 x 12 heads of 538, 360 blocks, 27 -> 29)
        const int rows = backward ? 128 : 32 * p.nw;
        const long blocks = (long)d->B * (backward ? (d->Hk < d->H ? d->Hk : d->H) : d->H) * ((d->Nq + rows - 1) / rows);
        p.ordered = blocks > 512 && p.ntq <= ORDER_TILES && p.ntk <= ORDER_TILES && p.ntq > 0 && p.ntk > 0 && p.nw != 1;
        if (p.ordered) { p.order_q = take(4l * d->B * ((d->Nq + rows - 1) / rows)); p.order_k = take(backward ? 4l * d->B * ((d->Nk + rows - 1) / rows) : 0); }
    }
    p.bytes = at;
    return p;
}

int mod_check(const mrg_attn_mod_desc* d, const char* who) {
    MRG_REQUIRE(d != nullptr, MRG_ERR_ARG, "%s: null descriptor", who);
    MRG_REQUIRE(d->head_dim == 32 || d->head_dim == 64, MRG_ERR_UNSUPPORTED, "%s: head_dim %d not in (32, 64)", who, d->head_dim);
    MRG_REQUIRE(d->B >= 0 && d->H > 0 && d->Hk > 0 && d->Nq >= 0 && d->Nk >= 0 && d->H % d->Hk == 0, MRG_ERR_SHAPE, "%s: bad sizes B %d H %d Hk %d Nq %d Nk %d", who,
                d->B, d->H, d->Hk, d->Nq, d->Nk);
    MRG_REQUIRE(d->Nq <= (1 << 26) && d->Nk <= (1 << 26) && (long)d->B * d->H * (((long)(d->Nq > d->Nk ? d->Nq : d->Nk) + 31) / 32) * MAX_SPLITS <= 0x7fffffffl,
                MRG_ERR_SHAPE, "%s: too many rows for one launch", who);
    const long steps[] = {d->q_bs, d->q_rs, d->q_hs, d->k_bs, d->k_rs, d->k_hs, d->v_bs, d->v_rs, d->v_hs, d->o_bs, d->o_rs, d->o_hs, d->do_bs, d->do_rs, d->do_hs,
                          d->dq_bs, d->dq_rs, d->dq_hs, d->dk_bs, d->dk_rs, d->dk_hs, d->dv_bs, d->dv_rs, d->dv_hs};
    for (const long s : steps) MRG_REQUIRE(s >= 0, MRG_ERR_SHAPE, "%s: negative stride %ld", who, s);
    // a tile's rows are addressed by 32-bit unsigned offsets from its first one
    MRG_REQUIRE((d->Nq <= 1 || (d->q_rs <= (1 << 23) && d->do_rs <= (1 << 23))) && (d->Nk <= 1 || (d->k_rs <= (1 << 23) && d->v_rs <= (1 << 23))), MRG_ERR_SHAPE, "%s: row strides above 2^23 elements", who);
    // (the kernels form scale / cap, slope / scale and lse / scale in fp32)
    MRG_REQUIRE(d->scale >= 1e-30f && d->scale < 1e30f, MRG_ERR_ARG, "%s: scale %g must be positive and finite (1e-30 to 1e30)", who, d->scale);
    MRG_REQUIRE(d->cap == 0.f || (d->cap >= 1e-30f && d->cap < 1e30f), MRG_ERR_ARG, "%s: cap %g must be 0 (none) or positive and finite (1e-30 to 1e30)", who, d->cap);
    MRG_REQUIRE(d->cap == 0.f || d->scale <= 1e30f * d->cap, MRG_ERR_ARG, "%s: cap %g is too small for a scale of %g", who, d->cap, d->scale);
    const bool some = d->B > 0 && d->Nq > 0 && d->Nk > 0;        // (tensors without elements may have no address)
    MRG_REQUIRE(!some || ((d->slopes != nullptr) == (d->pos_q != nullptr) && (d->slopes != nullptr) == (d->pos_k != nullptr)), MRG_ERR_ARG, "%s: a distance bias needs slopes, pos_q and pos_k", who);
    MRG_REQUIRE(!d->slopes || (d->axes >= 1 && d->axes <= MRG_MAX_AXES), MRG_ERR_SHAPE, "%s: %d axes (1 to %d)", who, d->axes, MRG_MAX_AXES);
    MRG_REQUIRE(!some || (d->doc_q != nullptr) == (d->doc_k != nullptr), MRG_ERR_ARG, "%s: documents of the queries and of the keys come together", who);
    MRG_REQUIRE(!d->prefix || d->causal, MRG_ERR_ARG, "%s: a prefix without causal order has no effect", who);
    return MRG_OK;
}

bool aligned8(const void* p, long a, long b, long c) { return (uintptr_t)p % 16 == 0 && (a | b | c) % 8 == 0; }

ModArgs mod_args(const mrg_attn_mod_desc* d, const Plan& p) {
    ModArgs a = {};
    a.q = (const bf16_t*)d->q; a.k = (const bf16_t*)d->k; a.v = (const bf16_t*)d->v; a.o = (bf16_t*)d->o; a.o_rest = (bf16_t*)d->o_rest; a.lse = d->lse;
    a.q_bs = d->q_bs; a.q_rs = d->q_rs; a.q_hs = d->q_hs; a.k_bs = d->k_bs; a.k_rs = d->k_rs; a.k_hs = d->k_hs;
    a.v_bs = d->v_bs; a.v_rs = d->v_rs; a.v_hs = d->v_hs; a.o_bs = d->o_bs; a.o_rs = d->o_rs; a.o_hs = d->o_hs;
    a.B = d->B; a.H = d->H; a.Hk = d->Hk; a.G = d->H / d->Hk; a.Nq = d->Nq; a.Nk = d->Nk; a.scale = d->scale; a.cap = d->cap;
    a.slopes = d->slopes; a.pos_q = d->pos_q; a.pos_k = d->pos_k; a.axes = d->slopes ? d->axes : 0;
    a.doc_q = d->doc_q; a.doc_k = d->doc_k;
    char* ws = (char*)d->ws;
    if (p.tables) { a.tab_q = (const int4*)(ws + p.tab_q); a.tab_k = (const int4*)(ws + p.tab_k); }
    a.ntq = p.ntq; a.ntk = p.ntk;
    a.causal = d->causal != 0; a.prefix = d->prefix;
    a.d_o = (const bf16_t*)d->d_o; a.do_bs = d->do_bs; a.do_rs = d->do_rs; a.do_hs = d->do_hs;
    a.dq = (bf16_t*)d->dq; a.dk = (bf16_t*)d->dk; a.dv = (bf16_t*)d->dv;
    a.dq_bs = d->dq_bs; a.dq_rs = d->dq_rs; a.dq_hs = d->dq_hs; a.dk_bs = d->dk_bs; a.dk_rs = d->dk_rs; a.dk_hs = d->dk_hs;
    a.dv_bs = d->dv_bs; a.dv_rs = d->dv_rs; a.dv_hs = d->dv_hs;
    a.dsum = (float*)(ws + p.dsum); a.part = (float*)(ws + p.part); a.part_ml = (float*)(ws + p.part_ml);
    return a;
}

void doc_tables(const mrg_attn_mod_desc* d, const Plan& p, ModArgs& a, bool backward, hipStream_t st) {
    if (!p.tables) return;
    const bool same = d->doc_q == d->doc_k && d->Nq == d->Nk;
    if (same) a.tab_q = a.tab_k;
    if (p.ordered) {
        char* ws = (char*)d->ws;
        const OrderArgs o = {d->doc_q, d->doc_k, (int4*)a.tab_q, (int4*)a.tab_k, (int*)(ws + p.order_q), backward ? (int*)(ws + p.order_k) : nullptr,
                             d->Nq, d->Nk, p.ntq, p.ntk, backward ? 128 : 32 * p.nw, d->causal != 0, d->prefix};
        hipLaunchKernelGGL(doc_order_kernel, dim3(d->B), dim3(ORDER_THREADS), 0, st, o);
        return;
    }
    const int ntq = same || !d->doc_q ? 0 : p.ntq, tiles = d->B * (ntq + p.ntk);
    if (tiles) hipLaunchKernelGGL(doc_tiles_kernel, dim3((tiles + 3) / 4), dim3(256), 0, st, d->doc_q, d->doc_k, (int4*)a.tab_q, (int4*)a.tab_k, d->B, d->Nq, d->Nk, ntq, p.ntk);
}

// Do the heads' blocks start side by side?  Where blocks differ in length the short ones then fill the end, and a CU's workgroups are not all of one
// length: under an order of the keys or of the blocks and with documents (one head after the other left a quarter of the chip idle behind the last
// head's long blocks; 4 x 12 heads of 1024 tokens in five documents 32 -> 28 us, 32 x 12 of them 113 -> 105), and where the last block holds one
// wave's rows or fewer, while what a die's heads read stays in its 4 MB of L2 (64 x 12 heads of 129 / 144 / 160 tokens: forward 30.3 -> 26.9,
// 29.7 -> 26.2, 30.0 -> 27.0 us, backward 78 -> 69, 78 -> 71, 79 -> 73; behind it two waves' rows gain less, 161 tokens 31 -> 29 and 84 -> 80, and
// where a die reads more they lose: 257 / 272 / 288 tokens, 6 MB, 48.7 -> 50.4, 51.2, 51.8; 16 x 12 heads of 1025 93 -> 97).  Split rows stay together.
bool start_abreast(const ModArgs& a, int rows, int heads, long head_bytes) {
    if (a.causal) return true;
    if (a.splits > 1) return false;
    const int tail = rows % 128;
    return a.tab_k != nullptr || (tail > 0 && tail <= 32 && (heads + 7) / 8 * head_bytes <= (4l << 20));
}

template <int HD, int NW, int CAP>
void fwd_go(const ModArgs& a, dim3 grid, hipStream_t st) {
    if (a.slopes) hipLaunchKernelGGL((attn_mod_fwd_kernel<HD, NW, CAP, true>), grid, dim3(64 * NW), 0, st, a);
    else hipLaunchKernelGGL((attn_mod_fwd_kernel<HD, NW, CAP, false>), grid, dim3(64 * NW), 0, st, a);
}
template <int HD, int NW>
void fwd_go(const ModArgs& a, dim3 grid, hipStream_t st) {
    if (a.cap > CAP_NEAR) fwd_go<HD, NW, FAR>(a, grid, st);
    else if (a.cap > 0.f) fwd_go<HD, NW, NEAR>(a, grid, st);
    else fwd_go<HD, NW, 0>(a, grid, st);
}
template <int HD, bool OWN_Q, int CAP>
void bwd_go(const ModArgs& a, dim3 grid, hipStream_t st) {
    if (a.slopes) hipLaunchKernelGGL((attn_mod_bwd_kernel<HD, OWN_Q, CAP, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((attn_mod_bwd_kernel<HD, OWN_Q, CAP, false>), grid, dim3(256), 0, st, a);
}
template <int HD, bool OWN_Q>
void bwd_go(const ModArgs& a, dim3 grid, hipStream_t st) {
    if (a.cap > CAP_NEAR) bwd_go<HD, OWN_Q, FAR>(a, grid, st);
    else if (a.cap > 0.f) bwd_go<HD, OWN_Q, NEAR>(a, grid, st);
    else bwd_go<HD, OWN_Q, 0>(a, grid, st);
}
template <bool OWN_Q>
void bwd_side(ModArgs a, int splits, int HD, hipStream_t st) {
    const int NO = OWN_Q ? a.Nq : a.Nk, OH = OWN_Q ? a.H : a.Hk;
    if (NO == 0) return;
    a.splits = splits;
    a.nblk = (NO + 127) / 128;
    a.abreast = start_abreast(a, NO, a.B * a.Hk, 4l * HD * (OWN_Q ? a.Nk : a.Nq * (long)a.G));
    // a launch has less than 2^32 threads along a dimension; a forward pass of up to 32 tokens a head fits more heads into them than these workgroups do
    const long blocks = (long)a.B * OH * a.nblk * splits, across = blocks < (1l << 24) ? blocks : 1l << 23;
    const dim3 grid((unsigned)across, (unsigned)((blocks + across - 1) / across));
    if (HD == 64) bwd_go<64, OWN_Q>(a, grid, st); else bwd_go<32, OWN_Q>(a, grid, st);
    if (splits > 1) {
        const long rows = (long)a.B * OH * NO, threads = rows * (OWN_Q ? 1 : 2) * HD / 4;
        const JoinOut o0 = OWN_Q ? JoinOut{a.dq, a.dq_bs, a.dq_rs, a.dq_hs} : JoinOut{a.dk, a.dk_bs, a.dk_rs, a.dk_hs}, o1 = JoinOut{a.dv, a.dv_bs, a.dv_rs, a.dv_hs};
        hipLaunchKernelGGL(attn_mod_sum_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, a.part, splits, rows, OWN_Q ? 1 : 2, HD, OH, NO, o0, o1);
    }
}

}  // namespace

extern "C" long mrg_attn_mod_ws_bytes(const mrg_attn_mod_desc* d, int backward) {
    if (mod_check(d, "mrg_attn_mod_ws_bytes")) return -1;
    return plan_for(d, backward != 0).bytes;
}

extern "C" int mrg_attn_mod_fwd(const mrg_attn_mod_desc* d, hipStream_t stream) {
    const int rc = mod_check(d, "mrg_attn_mod_fwd");
    if (rc) return rc;
    if (d->B == 0 || d->Nq == 0) return MRG_OK;
    const Plan p = plan_for(d, false);
    MRG_REQUIRE(d->q && d->o && (d->Nk == 0 || (d->k && d->v)) && (p.bytes == 0 || d->ws), MRG_ERR_ARG, "mrg_attn_mod_fwd: null pointer");
    MRG_REQUIRE(aligned8(d->q, d->q_bs, d->q_rs, d->q_hs) && aligned8(d->k, d->k_bs, d->k_rs, d->k_hs) && aligned8(d->v, d->v_bs, d->v_rs, d->v_hs)
                && aligned8(d->o, d->o_bs, d->o_rs, d->o_hs) && (uintptr_t)d->o_rest % 16 == 0, MRG_ERR_ARG, "mrg_attn_mod_fwd: operands and their strides must be multiples of 16 bytes");
    ModArgs a = mod_args(d, p);
    a.nblk = p.nblk; a.splits = p.splits;
    if (p.ordered) a.order = (const int*)((char*)d->ws + p.order_q);
    a.abreast = start_abreast(a, a.Nq, a.B * a.Hk, 4l * d->head_dim * a.Nk);
    doc_tables(d, p, a, false, stream);
    const dim3 grid((unsigned)((long)a.B * a.H * a.nblk * a.splits));
    if (d->head_dim == 64) { if (p.nw == 1) fwd_go<64, 1>(a, grid, stream); else fwd_go<64, 4>(a, grid, stream); }
    else { if (p.nw == 1) fwd_go<32, 1>(a, grid, stream); else fwd_go<32, 4>(a, grid, stream); }
    if (a.splits > 1) {
        const dim3 rows((unsigned)(((long)a.B * a.H * a.Nq + 3) / 4));
        if (d->head_dim == 64) hipLaunchKernelGGL(attn_mod_join_kernel<64>, rows, dim3(256), 0, stream, a);
        else hipLaunchKernelGGL(attn_mod_join_kernel<32>, rows, dim3(256), 0, stream, a);
    }
    return mrg_check_launch("mrg_attn_mod_fwd");
}

extern "C" int mrg_attn_mod_bwd(const mrg_attn_mod_desc* d, hipStream_t stream) {
    const int rc = mod_check(d, "mrg_attn_mod_bwd");
    if (rc) return rc;
    if (d->B == 0 || (d->Nq == 0 && d->Nk == 0)) return MRG_OK;
    const Plan p = plan_for(d, true);
    MRG_REQUIRE((d->Nq == 0 || (d->q && d->o && d->lse && d->d_o && d->dq)) && (d->Nk == 0 || (d->k && d->v && d->dk && d->dv)) && (p.bytes == 0 || d->ws), MRG_ERR_ARG,
                "mrg_attn_mod_bwd: null pointer");
    MRG_REQUIRE(aligned8(d->q, d->q_bs, d->q_rs, d->q_hs) && aligned8(d->k, d->k_bs, d->k_rs, d->k_hs) && aligned8(d->v, d->v_bs, d->v_rs, d->v_hs)
                && aligned8(d->o, d->o_bs, d->o_rs, d->o_hs) && (uintptr_t)d->o_rest % 16 == 0 && aligned8(d->d_o, d->do_bs, d->do_rs, d->do_hs) && aligned8(d->dq, d->dq_bs, d->dq_rs, d->dq_hs)
                && aligned8(d->dk, d->dk_bs, d->dk_rs, d->dk_hs) && aligned8(d->dv, d->dv_bs, d->dv_rs, d->dv_hs), MRG_ERR_ARG,
                "mrg_attn_mod_bwd: operands and their strides must be multiples of 16 bytes");
    ModArgs a = mod_args(d, p);
    doc_tables(d, p, a, true, stream);
    if (p.ordered) a.order = (const int*)((char*)d->ws + p.order_q);
    bwd_side<true>(a, p.dq_splits, d->head_dim, stream);
    if (p.ordered) a.order = (const int*)((char*)d->ws + p.order_k);
    bwd_side<false>(a, p.dkv_splits, d->head_dim, stream);
    return mrg_check_launch("mrg_attn_mod_bwd");
}
