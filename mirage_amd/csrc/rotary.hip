// Rotary positions with several axes (stack, height, width): every pair (a, b) of a head's leading 2 P elements is turned by
//     theta[row, p] = pos[row, axis(p)] * freqs[p]          (a, b) -> (a cos - b sin, a sin + b cos)
// for q and k in one launch; `inverse` turns by -theta, which is also the gradient (a rotation's transpose is its inverse).
//
// The angle is reduced in 64 bits: it is formed in turns (pos * freq / 2 pi), its nearest whole number is taken off, and what is left, at most
// half a turn, goes to fp32 with an absolute error of 2^-26 turns.  In fp32 a position of 10^6 alone would lose 0.06 rad.  Sine and cosine of
// a (row, pair) are computed once per workgroup into LDS and shared by all its heads: at 12 - 16 heads the 64-bit arithmetic fits into the
// issue slots that the copy of the row leaves free.
//
// Bound: HBM, one read and one write of q and k: 8 x 4097 rows of 16 + 16 heads of 64 in bf16 take 50 us a turn, 5.3 TB/s (a plain copy of 2 GiB ran at
// 4.9); a single image (257 rows of 12 + 12 heads) 3.1 us, which is a launch.  A workgroup owns `rows` whole rows of q or of k (blockIdx.y), walks
// their (head, 8 pairs) units with 16-byte loads of both members of the pairs (bf16; 4 pairs in fp32) and keeps ROT_UNITS units in flight per
// lane before it stores the first.
#include "common.h"
#include "mirage_hip.h"

namespace {

constexpr int ROT_UNITS = 2;       // units in flight per lane (4 the same on long rows, 5 % slower on small ones: their registers cost waves)
constexpr int ROT_MAX_HD = 256;

struct RotSide { const char* in; char* out; long bs, rs, hs, obs, ors, ohs; int H; };
struct RotArgs {
    RotSide s[2];                  // q, k
    const void* pos; long pos_bs, pos_rs; int pos_f32;
    const double* freqs;
    int N, P, cut0, cut1;          // pairs of axis 0 / axes 0 and 1 end here
    int axial, dist;               // half: second = first + dist; axial: the axis' own width
    int units, tail;               // rotated units and copied units (elements behind the pairs) per head
    int rows_total, rows;          // rows per workgroup
    float sign;
};

template <typename T, int VEC> struct Pack { T v[VEC]; };
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> rot_load(const T* p) { return *reinterpret_cast<const Pack<T, VEC>*>(__builtin_assume_aligned(p, sizeof(T) * VEC)); }
template <typename T, int VEC>
__device__ __forceinline__ void rot_store(T* p, const Pack<T, VEC>& v) { *reinterpret_cast<Pack<T, VEC>*>(__builtin_assume_aligned(p, sizeof(T) * VEC)) = v; }
__device__ __forceinline__ float rot_f(float x) { return x; }
__device__ __forceinline__ float rot_f(bf16_t x) { return bf2f(x); }
__device__ __forceinline__ void rot_put(float& d, float x) { d = x; }
__device__ __forceinline__ void rot_put(bf16_t& d, float x) { d = f2bf(x); }

// VEC pairs of a unit: halves -> VEC first members at `lo`, VEC second members at `hi`; interleaved -> 2 VEC elements at `lo`, hi = lo + VEC
template <typename T, int VEC, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(const RotArgs a) {
    extern __shared__ __attribute__((aligned(16))) float2 cs[];        // [rows][P] (cos, sin)
    const unsigned start = (blockIdx.z * gridDim.x + blockIdx.x) * a.rows;     // (a further dimension from 2^24 workgroups on)
    if (start >= (unsigned)a.rows_total) return;
    const int r0 = (int)start, nrow = min(a.rows, a.rows_total - r0);
    const int P = a.P;
    for (int i = threadIdx.x; i < nrow * P; i += 256) {
        const int rr = i / P, p = i - rr * P;
        const int row = r0 + rr, b = row / a.N, n = row - b * a.N;
        const int ax = (p >= a.cut0) + (p >= a.cut1);
        const long at = (long)b * a.pos_bs + (long)n * a.pos_rs + ax;
        const double x = a.pos_f32 ? (double)reinterpret_cast<const float*>(a.pos)[at] : (double)reinterpret_cast<const int*>(a.pos)[at];
        double t = x * (a.freqs[p] * 0.15915494309189533577);          // turns
        t -= rint(t);
        float s, c;
        sincospif(2.0f * (float)t, &s, &c);
        cs[i] = make_float2(c, a.sign * s);
    }
    __syncthreads();
    const RotSide s = a.s[blockIdx.y];
    const int per_head = a.units + a.tail, per_row = s.H * per_head, total = nrow * per_row;
    for (int i0 = threadIdx.x; i0 < total; i0 += 256 * ROT_UNITS) {
        Pack<T, VEC> lo[ROT_UNITS], hi[ROT_UNITS];
        T* dlo[ROT_UNITS];
        int off2[ROT_UNITS], ci[ROT_UNITS];                            // distance to the second vector (0: a copied unit), index into cs
#pragma unroll
        for (int j = 0; j < ROT_UNITS; ++j) {
            const int i = i0 + 256 * j;
            dlo[j] = nullptr;
            if (i < total) {
                const int rr = i / per_row, w = i - rr * per_row;
                const int h = w / per_head, u = w - h * per_head;
                const int row = r0 + rr, b = row / a.N, n = row - b * a.N;
                int e, d2 = 0;
                if (u >= a.units) e = 2 * P + (u - a.units) * VEC;
                else if (INTER) { e = 2 * u * VEC; d2 = VEC; }
                else {
                    const int p = u * VEC;
                    e = p; d2 = a.dist;
                    if (a.axial) {
                        const int ax = (p >= a.cut0) + (p >= a.cut1);
                        const int start = ax == 0 ? 0 : (ax == 1 ? a.cut0 : a.cut1);
                        d2 = (ax == 0 ? a.cut0 : (ax == 1 ? a.cut1 - a.cut0 : P - a.cut1));
                        e = p + start;
                    }
                }
                const T* src = reinterpret_cast<const T*>(s.in) + (long)b * s.bs + (long)n * s.rs + (long)h * s.hs + e;
                dlo[j] = reinterpret_cast<T*>(s.out) + (long)b * s.obs + (long)n * s.ors + (long)h * s.ohs + e;
                off2[j] = d2;
                ci[j] = rr * P + u * VEC;
                lo[j] = rot_load<T, VEC>(src);
                if (d2) hi[j] = rot_load<T, VEC>(src + d2);
            }
        }
#pragma unroll
        for (int j = 0; j < ROT_UNITS; ++j) {
            if (dlo[j] == nullptr) continue;
            if (off2[j]) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float2 c = cs[ci[j] + e];
                    T& ra = INTER ? (2 * e < VEC ? lo[j].v[(2 * e) % VEC] : hi[j].v[(2 * e) % VEC]) : lo[j].v[e];
                    T& rb = INTER ? (2 * e + 1 < VEC ? lo[j].v[(2 * e + 1) % VEC] : hi[j].v[(2 * e + 1) % VEC]) : hi[j].v[e];
                    const float x = rot_f(ra), y = rot_f(rb);
                    rot_put(ra, x * c.x - y * c.y);
                    rot_put(rb, x * c.y + y * c.x);
                }
                rot_store<T, VEC>(dlo[j] + off2[j], hi[j]);
            }
            rot_store<T, VEC>(dlo[j], lo[j]);
        }
    }
}

template <typename T, int VEC>
void rot_launch(const RotArgs& a, bool inter, dim3 grid, size_t lds, hipStream_t st) {
    if (inter) hipLaunchKernelGGL((rotary_kernel<T, VEC, true>), grid, dim3(256), lds, st, a);
    else hipLaunchKernelGGL((rotary_kernel<T, VEC, false>), grid, dim3(256), lds, st, a);
}

}  // namespace

extern "C" int mrg_rotary_axes(const mrg_rotary_desc* d, hipStream_t stream) {
    MRG_REQUIRE(d != nullptr, MRG_ERR_ARG, "mrg_rotary_axes: null descriptor");
    MRG_REQUIRE(d->dtype == MRG_DT_BF16 || d->dtype == MRG_DT_F32, MRG_ERR_ARG, "mrg_rotary_axes: dtype %d is neither bf16 nor fp32", d->dtype);
    MRG_REQUIRE(d->pos_dtype == MRG_POS_I32 || d->pos_dtype == MRG_POS_F32, MRG_ERR_ARG, "mrg_rotary_axes: positions are int32 or fp32");
    MRG_REQUIRE(d->pairing >= MRG_PAIR_HALF && d->pairing <= MRG_PAIR_AXIAL, MRG_ERR_ARG, "mrg_rotary_axes: unknown pairing %d", d->pairing);
    MRG_REQUIRE(d->axes >= 1 && d->axes <= MRG_MAX_AXES, MRG_ERR_SHAPE, "mrg_rotary_axes: %d axes (1 to %d)", d->axes, MRG_MAX_AXES);
    MRG_REQUIRE(d->B >= 0 && d->N >= 0 && d->Hq >= 0 && d->Hk >= 0, MRG_ERR_SHAPE, "mrg_rotary_axes: negative size");
    MRG_REQUIRE(d->head_dim >= 2 && d->head_dim <= ROT_MAX_HD, MRG_ERR_SHAPE, "mrg_rotary_axes: head_dim %d (2 to %d)", d->head_dim, ROT_MAX_HD);
    int P = 0, cut[MRG_MAX_AXES];
    for (int i = 0; i < MRG_MAX_AXES; ++i) {
        const int w = i < d->axes ? d->sections[i] : 0;
        MRG_REQUIRE(w >= 0 && (i >= d->axes || w > 0) && w <= d->head_dim, MRG_ERR_SHAPE, "mrg_rotary_axes: section %d has %d pairs", i, w);
        P += w;
        cut[i] = P;
    }
    MRG_REQUIRE(2 * P <= d->head_dim, MRG_ERR_SHAPE, "mrg_rotary_axes: %d pairs do not fit a head of %d", P, d->head_dim);
    if (d->B == 0 || d->N == 0 || d->Hq + d->Hk == 0) return MRG_OK;
    MRG_REQUIRE((long)d->B * d->N <= 0x7fffffffl - 1024 && (long)(d->Hq + d->Hk) * d->head_dim <= (1 << 24), MRG_ERR_SHAPE, "mrg_rotary_axes: too many rows or heads");
    MRG_REQUIRE(d->pos && d->freqs && (d->Hq == 0 || (d->q && d->q_out)) && (d->Hk == 0 || (d->k && d->k_out)), MRG_ERR_ARG, "mrg_rotary_axes: null pointer");
    RotArgs a;
    int sides = 0;
    if (d->Hq) a.s[sides++] = {(const char*)d->q, (char*)d->q_out, d->q_bs, d->q_rs, d->q_hs, d->qo_bs, d->qo_rs, d->qo_hs, d->Hq};
    if (d->Hk) a.s[sides++] = {(const char*)d->k, (char*)d->k_out, d->k_bs, d->k_rs, d->k_hs, d->ko_bs, d->ko_rs, d->ko_hs, d->Hk};
    a.pos = d->pos; a.pos_bs = d->pos_bs; a.pos_rs = d->pos_rs; a.pos_f32 = d->pos_dtype == MRG_POS_F32;
    a.freqs = d->freqs;
    a.N = d->N; a.P = P;
    a.cut0 = cut[0]; a.cut1 = cut[1];
    a.axial = d->pairing == MRG_PAIR_AXIAL;
    a.dist = P;
    a.sign = d->inverse ? -1.f : 1.f;
    a.rows_total = d->B * d->N;
    const bool inter = d->pairing == MRG_PAIR_INTERLEAVED;
    // widest unit (16 bytes down to one element) that every span, stride and pointer allows
    const int size = d->dtype == MRG_DT_BF16 ? 2 : 4;
    int vec = 16 / size;
    auto fits = [&](int v) {
        unsigned long bits = (unsigned long)(d->head_dim - 2 * P);
        if (a.axial) for (int i = 0; i < d->axes; ++i) bits |= (unsigned long)d->sections[i];
        else bits |= (unsigned long)P;
        for (int i = 0; i < sides; ++i) {
            const RotSide& s = a.s[i];
            bits |= (unsigned long)(s.bs | s.rs | s.hs | s.obs | s.ors | s.ohs);
            if (((uintptr_t)s.in | (uintptr_t)s.out) % (size_t)(v * size)) return false;
        }
        return bits % (unsigned long)v == 0;
    };
    while (vec > 1 && !fits(vec)) vec >>= 1;
    MRG_REQUIRE(fits(1), MRG_ERR_ARG, "mrg_rotary_axes: pointers are not aligned to their element");
    a.units = P / vec;
    bool copy = false;                                        // elements behind the pairs are copied unless both sides work in place
    for (int i = 0; i < sides; ++i) copy |= a.s[i].in != a.s[i].out;
    a.tail = copy ? (d->head_dim - 2 * P) / vec : 0;
    // rows of a workgroup: enough workgroups for every CU first (one row each: a single image is a latency matter), then rows until every lane has a
    // unit.  Forward and back at 32776 rows x 32 heads of 64 (64 units a row): 161 us with one row, 101 with 4, 105 with 8, 108 with 16;
    // 16512 rows x 12 heads (24 units): 15 us with 4 rows, 12 with 8 and with 16
    int rows = 1;
    const int row_units = (a.s[0].H > a.s[sides - 1].H ? a.s[0].H : a.s[sides - 1].H) * (a.units + a.tail);
    while (rows < 16 && rows * row_units < 256 && a.rows_total / rows > 2048) rows <<= 1;
    a.rows = rows;
    // a launch has less than 2^32 threads along a dimension
    const int blocks = (a.rows_total + rows - 1) / rows, across = blocks < (1 << 24) ? blocks : 1 << 23;
    const dim3 grid(across, sides, (blocks - 1) / across + 1);
    const size_t lds = sizeof(float2) * rows * P;
    if (d->dtype == MRG_DT_BF16) {
        if (vec == 8) rot_launch<bf16_t, 8>(a, inter, grid, lds, stream);
        else if (vec == 4) rot_launch<bf16_t, 4>(a, inter, grid, lds, stream);
        else if (vec == 2) rot_launch<bf16_t, 2>(a, inter, grid, lds, stream);
        else rot_launch<bf16_t, 1>(a, inter, grid, lds, stream);
    } else {
        if (vec == 4) rot_launch<float, 4>(a, inter, grid, lds, stream);
        else if (vec == 2) rot_launch<float, 2>(a, inter, grid, lds, stream);
        else rot_launch<float, 1>(a, inter, grid, lds, stream);
    }
    return mrg_check_launch("mrg_rotary_axes");
}
