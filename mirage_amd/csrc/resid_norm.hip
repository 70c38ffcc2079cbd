// The seam between two branches of a block in one pass: norm behind a branch, gate, scaled residual, norm in front of the next branch.
//     n = Norm_post(branch)     x' = alpha x + gate * n     y = Norm_pre(x')          Norm: layer (mean and variance) or rms
// gate is absent, one row of channels, or one row per sample; either norm may be absent.  With xhat, bhat the normalised rows and r the
// reciprocal deviations, the gradient is
//     t       = dx' + r_pre (dy w_pre - mean(dy w_pre) - xhat mean(dy w_pre xhat))          (rms: without the first mean)
//     dx      = alpha t
//     dbranch = r_post (g t w_post - mean(g t w_post) - bhat mean(g t w_post bhat))         (no post norm: g t)
//     dw_pre  = sum dy xhat    db_pre = sum dy
// and everything else follows from the two column sums A = sum t bhat and T = sum t over the rows that share a gate:
//     dgate = w_post A + b_post T      dw_post = sum over gates of g A      db_post = sum over gates of g T
// so a workgroup carries four sums per column instead of five, whatever the gate's shape.
//
// Bound: HBM.  Forward reads 4 + 2 and writes 4 + 2 bytes an element (fp32 residual, bf16 branch and y), backward reads 12 and writes 6: 65792
// rows of 1024 with a gate per sample take 182 us (4.4 TB/s) and 258 us (4.7 TB/s, the adding of the partial sums with it), where a plain copy of
// 2 GiB ran at 4.9.
// A row is read once into registers (forward: a wave per row up to 1024 columns, four waves beyond; backward, which carries the column sums
// and a requested row as well: one wave per 256 columns), all statistics in fp32: the mean first, then the
// squares of the differences, from registers.  Column sums stay in registers over a workgroup's rows, meet in LDS, and leave as one
// partial row per workgroup that a second launch adds in a fixed order: no atomics, the same bits on every run.
#include "common.h"
#include "mirage_hip.h"

namespace {

struct ResidArgs {
    const float* x; const void* branch; const float* gate; long gate_stride; float alpha;
    const float* post_w; const float* post_b; const float* pre_w; const float* pre_b;
    float* x_new; void* y; int y_f32; float* stats;      // stats [4][M]: post mean, post rstd, pre mean, pre rstd
    int M, L, D, layer; float eps;                        // L: rows that share a gate
    // backward
    const float* dx_new; const void* dy; int dy_f32, branch_f32; float* dx; void* dbranch;
    float* part;                                          // [grid][4][D]: dw_pre, db_pre, dw_post (or dgate), db_post
    float* gpart;                                         // [samples * parts][D] dgate of each unit
    int parts, units;
};

__device__ __forceinline__ float4 rn_bf4(uint2 u) {
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ float4 rn_load(const void* p, long row, int D, int c, bool f32) {
    if (f32) return reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + row * D)[c];
    return rn_bf4(reinterpret_cast<const uint2*>(reinterpret_cast<const bf16_t*>(p) + row * D)[c]);
}
// the same without opening bf16 (a requested row waits in the form it came in)
__device__ __forceinline__ float4 rn_raw(const void* p, long row, int D, int c, bool f32) {
    if (f32) return reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + row * D)[c];
    const uint2 u = reinterpret_cast<const uint2*>(reinterpret_cast<const bf16_t*>(p) + row * D)[c];
    return make_float4(__uint_as_float(u.x), __uint_as_float(u.y), 0.f, 0.f);
}
__device__ __forceinline__ float4 rn_open(const float4 v, bool f32) { return f32 ? v : rn_bf4(make_uint2(__float_as_uint(v.x), __float_as_uint(v.y))); }
__device__ __forceinline__ void rn_store(void* p, long row, int D, int c, bool f32, const float4 v) {
    if (f32) reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + row * D)[c] = v;
    else reinterpret_cast<uint2*>(reinterpret_cast<bf16_t*>(p) + row * D)[c] = make_uint2(pack_bf2(v.x, v.y), pack_bf2(v.z, v.w));
}
__device__ __forceinline__ float sum4(const float4 a) { return (a.x + a.y) + (a.z + a.w); }
__device__ __forceinline__ float dot4(const float4 a, const float4 b) { return (a.x * b.x + a.y * b.y) + (a.z * b.z + a.w * b.w); }
__device__ __forceinline__ float4 operator*(const float4 a, const float4 b) { return make_float4(a.x * b.x, a.y * b.y, a.z * b.z, a.w * b.w); }
__device__ __forceinline__ float4 operator+(const float4 a, const float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
__device__ __forceinline__ float4 scale4(const float4 a, const float s) { return make_float4(a.x * s, a.y * s, a.z * s, a.w * s); }
__device__ __forceinline__ float4 shift4(const float4 a, const float s) { return make_float4(a.x - s, a.y - s, a.z - s, a.w - s); }
__device__ __forceinline__ float4 zero4() { return make_float4(0.f, 0.f, 0.f, 0.f); }
__device__ __forceinline__ float4 fma4(const float4 a, const float s, const float4 b) {
    return make_float4(fmaf(a.x, s, b.x), fmaf(a.y, s, b.y), fmaf(a.z, s, b.z), fmaf(a.w, s, b.w));
}

// sum over the lanes of a row: its wave, or its WPR waves through `box` (two alternating sets of slots; every wave of the workgroup calls it
// the same number of times)
template <int WPR>
struct RowSum {
    float (*box)[2][WPR]; int turn = 0, wave;
    __device__ __forceinline__ float2 operator()(float a, float b) {
        a = wave_sum(a); b = wave_sum(b);
        if (WPR == 1) return make_float2(a, b);
        float (&slot)[2][WPR] = box[turn];
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) { slot[0][wave] = a; slot[1][wave] = b; }
        __syncthreads();
        float2 s = make_float2(slot[0][0], slot[1][0]);
#pragma unroll
        for (int w = 1; w < WPR; ++w) { s.x += slot[0][w]; s.y += slot[1][w]; }
        return s;
    }
};

// mean (layer) and reciprocal deviation of the row whose chunks are v[]; columns outside the row hold zero in v and are skipped
template <int NV, int WPR>
__device__ __forceinline__ void row_stats(const float4 (&v)[NV], const bool (&ok)[NV], RowSum<WPR>& sum, float invD, int layer, float eps, float& mu, float& rs) {
    mu = 0.f;
    if (layer) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) s += sum4(v[j]);
        mu = sum(s, 0.f).x * invD;
    }
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) if (ok[j]) { const float4 d = shift4(v[j], mu); q += dot4(d, d); }
    rs = rsqrtf(sum(q, 0.f).x * invD + eps);
}

template <int NV, int WPR, bool BR32>
__global__ __launch_bounds__(256) void resid_norm_fwd_kernel(const ResidArgs a) {
    __shared__ float box[2][2][WPR];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned blk = blockIdx.y * gridDim.x + blockIdx.x;     // (a second dimension from 2^24 workgroups on)
    const unsigned at = WPR == 1 ? blk * 4 + wave : blk;
    if (at >= (unsigned)a.M) return;
    const int row = (int)at;
    RowSum<WPR> sum{box, 0, wave};
    const int D = a.D, nv = D >> 2, c0 = WPR == 1 ? lane : threadIdx.x, step = 64 * WPR;
    const float invD = 1.f / (float)D;
    const float4* gate = a.gate ? reinterpret_cast<const float4*>(a.gate + (long)(row / a.L) * a.gate_stride) : nullptr;
    float4 x[NV], n[NV], pw[NV], pb[NV];
    bool ok[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = c0 + step * j;
        ok[j] = c < nv;
        x[j] = n[j] = pw[j] = pb[j] = zero4();
        if (ok[j]) {
            x[j] = rn_load(a.x, row, D, c, true);
            n[j] = rn_load(a.branch, row, D, c, BR32);
            if (a.pre_w) pw[j] = reinterpret_cast<const float4*>(a.pre_w)[c];
            if (a.pre_b) pb[j] = reinterpret_cast<const float4*>(a.pre_b)[c];
        }
    }
    float mu, rs;
    if (a.post_w) {
        row_stats<NV, WPR>(n, ok, sum, invD, a.layer, a.eps, mu, rs);
        if (c0 == 0) { a.stats[row] = mu; a.stats[(long)a.M + row] = rs; }
#pragma unroll
        for (int j = 0; j < NV; ++j) if (ok[j]) {
            const int c = c0 + step * j;
            n[j] = scale4(shift4(n[j], mu), rs) * reinterpret_cast<const float4*>(a.post_w)[c];
            if (a.post_b) n[j] = n[j] + reinterpret_cast<const float4*>(a.post_b)[c];
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) if (ok[j]) {
        const int c = c0 + step * j;
        if (gate) n[j] = n[j] * gate[c];
        x[j] = fma4(x[j], a.alpha, n[j]);
        rn_store(a.x_new, row, D, c, true, x[j]);
    }
    if (!a.pre_w) return;
    row_stats<NV, WPR>(x, ok, sum, invD, a.layer, a.eps, mu, rs);
    if (c0 == 0) { a.stats[2l * a.M + row] = mu; a.stats[3l * a.M + row] = rs; }
#pragma unroll
    for (int j = 0; j < NV; ++j) if (ok[j]) rn_store(a.y, row, D, c0 + step * j, a.y_f32, scale4(shift4(x[j], mu), rs) * pw[j] + pb[j]);
}

// One float4 of a row per lane, WPR waves per row (WPR = 1: four rows side by side).  SAMPLE: a gate per sample -- the sums A and T are closed at the
// end of every unit (a part of one sample's rows) into gpart and into the workgroup's own dw_post / db_post; otherwise there is one gate (or none)
// and they are closed once
template <int WPR, bool POST, bool SAMPLE, bool PRE, bool B32, bool DY32>
__global__ __launch_bounds__(WPR == 1 ? 256 : 64 * WPR, 4) void resid_norm_bwd_kernel(const ResidArgs a) {
    __shared__ float box[2][2][WPR];
    __shared__ __attribute__((aligned(16))) float buf[WPR == 1 ? 4 * 256 : 4];
    const int wave = threadIdx.x >> 6;
    RowSum<WPR> sum{box, 0, wave};
    const int D = a.D, c = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
    const float invD = 1.f / (float)D;
    const bool ok = c < (D >> 2);
    const int cc = ok ? c : 0;                                    // lanes behind the row read its first chunk and count for nothing
    auto vec = [&](const float* p) { return p && ok ? reinterpret_cast<const float4*>(p)[c] : zero4(); };
    const float4 pre_w = vec(PRE ? a.pre_w : nullptr), post_w = vec(POST ? a.post_w : nullptr);
    float4 g = make_float4(1.f, 1.f, 1.f, 1.f);
    if (!SAMPLE && a.gate) g = vec(a.gate);
    float4 sw = zero4(), sb = zero4(), A = zero4(), T = zero4(), GA = zero4(), GT = zero4();
    // one column sum of the workgroup: its waves' registers meet in LDS (a wave per row) or are whole already
    auto flush = [&](const float4 v, float* out) {
        if (WPR == 1) {
            __syncthreads();
            if (ok) reinterpret_cast<float4*>(buf + wave * 256)[c] = v;
            __syncthreads();
            for (int i = threadIdx.x; i < D; i += 256) out[i] = (buf[i] + buf[256 + i]) + (buf[512 + i] + buf[768 + i]);
        } else if (ok) reinterpret_cast<float4*>(out)[c] = v;
    };
    // end of the rows that share a gate: dgate = w_post A + b_post T, and g A, g T towards dw_post, db_post
    auto close = [&](int slot) {
        if (a.gpart) {
            float4 dg = POST ? A * post_w : A;
            if (POST && a.post_b) dg = dg + T * vec(a.post_b);
            flush(dg, a.gpart + (long)slot * D);
        }
        GA = GA + A * g; GT = GT + T * g;
        if (SAMPLE) A = T = zero4();
    };
    const int u0 = (int)((long)blockIdx.x * a.units / gridDim.x), u1 = (int)((long)(blockIdx.x + 1) * a.units / gridDim.x);
    for (int u = u0; u < u1; ++u) {
        const int smp = u / a.parts, part = u - smp * a.parts;
        const int lo = smp * a.L + (int)((long)part * a.L / a.parts), hi = smp * a.L + (int)((long)(part + 1) * a.L / a.parts);
        if (SAMPLE) g = vec(a.gate + (long)smp * a.gate_stride);
        constexpr int RSTEP = WPR == 1 ? 4 : 1;
        const int first = lo + (WPR == 1 ? wave : 0);
        // the next row is requested before this one's sums and stores
        float4 nt = zero4(), nw = zero4(), nx = zero4(), nb = zero4(), nstat = zero4();
        auto fetch = [&](int row) {
            nt = rn_load(a.dx_new, row, D, cc, true);
            nb = rn_raw(a.branch, row, D, cc, B32);
            if (PRE) { nw = rn_raw(a.dy, row, D, cc, DY32); nx = rn_load(a.x_new, row, D, cc, true); }
            if (POST) { nstat.x = a.stats[row]; nstat.y = a.stats[(long)a.M + row]; }
            if (PRE) { nstat.z = a.stats[2l * a.M + row]; nstat.w = a.stats[3l * a.M + row]; }
        };
        if (first < hi) fetch(first);
        for (int row = first; row < hi; row += RSTEP) {
            float4 t = nt, b = rn_open(nb, B32), w = rn_open(nw, DY32), xh = nx;
            const float4 stat = nstat;
            if (!ok) t = b = w = xh = zero4();
            if (row + RSTEP < hi) fetch(row + RSTEP);
            if (PRE) {
                if (ok) xh = scale4(shift4(xh, stat.z), stat.w);
                sw = sw + w * xh;
                sb = sb + w;
                w = w * pre_w;
                const float2 m = sum(sum4(w), dot4(w, xh));
                const float m1 = a.layer ? m.x * invD : 0.f, m2 = m.y * invD;
                t = fma4(fma4(xh, -m2, shift4(w, m1)), stat.w, t);
            }
            if (POST && ok) b = scale4(shift4(b, stat.x), stat.y);
            if (ok) rn_store(a.dx, row, D, c, true, scale4(t, a.alpha));
            else t = zero4();
            A = A + t * b;
            if (POST) T = T + t;
            t = t * g;
            if (POST) {
                t = t * post_w;
                const float2 m = sum(sum4(t), dot4(t, b));
                const float m1 = a.layer ? m.x * invD : 0.f, m2 = m.y * invD;
                t = scale4(fma4(b, -m2, shift4(t, m1)), stat.y);
            }
            if (ok) rn_store(a.dbranch, row, D, c, B32, t);
        }
        if (SAMPLE) close(u);
    }
    if (!SAMPLE) close(blockIdx.x);
    float* out = a.part + (long)blockIdx.x * 4 * D;
    if (PRE) { flush(sw, out); if (a.pre_b) flush(sb, out + D); }
    if (POST) { flush(GA, out + 2 * D); if (a.post_b) flush(GT, out + 3 * D); }
}

// column sums of the partial rows: a job adds `n` rows that lie `stride` floats apart.  32 columns and 32 rows at a time; the order of the
// additions is fixed by the sizes alone.  More gates than a launch has workgroups for (2^24) are walked
struct SumJob { const float* src; float* dst; int n; long stride; };
struct SumArgs { SumJob job[4]; const float* gsrc; float* gdst; int parts, D, njobs, jobs; };
__global__ __launch_bounds__(256) void resid_norm_sum_kernel(const SumArgs a) {
    __shared__ __attribute__((aligned(16))) float4 box[32][8];
    const int cl = threadIdx.x & 7, rl = threadIdx.x >> 3;
    const int c = blockIdx.y * 8 + cl;
    for (long j = blockIdx.x; j < a.jobs; j += gridDim.x) {
        SumJob job;
        if (j < a.njobs) job = a.job[j];
        else {
            const long s = j - a.njobs;                     // one sample's gate: its parts are consecutive rows
            job = SumJob{a.gsrc + s * a.parts * a.D, a.gdst + s * a.D, a.parts, (long)a.D};
        }
        float4 s = zero4();
        if (c * 4 < a.D) {
#pragma unroll 4
            for (int r = rl; r < job.n; r += 32) s = s + reinterpret_cast<const float4*>(job.src + (long)r * job.stride)[c];
        }
        box[rl][cl] = s;
        __syncthreads();
        for (int w = 16; w > 0; w >>= 1) {
            if (rl < w) box[rl][cl] = box[rl][cl] + box[rl + w][cl];
            __syncthreads();
        }
        if (rl == 0 && c * 4 < a.D) reinterpret_cast<float4*>(job.dst)[c] = box[0][cl];      // (written again by this thread itself)
    }
}

// waves of a backward row, and of a workgroup (four rows side by side where one wave holds a row)
int rn_waves(int D) { return D <= 256 ? 1 : (D <= 512 ? 2 : (D <= 768 ? 3 : (D <= 1024 ? 4 : (D <= 2048 ? 8 : 16)))); }
// The backward launch: 12 of the 16 waves per CU that its registers allow, but a workgroup for every CU.  More of them leave more partial sums (65792 x
// 1024, forward and backward: 455 us with 16 waves, 440 with 12; 8200 x 4096, backward: 203 us with four workgroups per CU, 147 with one), fewer
// keep too little in flight (16448 x 512: 34 us with 12, 39 with 8, 44 with 4).
// Units: the rows that share a gate, cut into parts until every workgroup has one, but no part below 16 rows (four per wave) where a gate has that
// many; more units than workgroups fit at once are dealt evenly.
int rn_groups(int D, int waves_per_cu) { const int w = rn_waves(D), n = waves_per_cu / (w == 1 ? 4 : w); return 256 * (n < 1 ? 1 : n); }
int rn_parts(int samples, int L, int D) {
    const int parts = (rn_groups(D, 12) + samples - 1) / samples, most = (L + 15) / 16;
    return parts < 1 ? 1 : (parts > most ? (most < 1 ? 1 : most) : parts);
}
int rn_grid(long units, int D) {
    const long fit = rn_groups(D, 16), each = (units + fit - 1) / fit;
    return (int)((units + each - 1) / each);
}

template <int WPR, bool B32, bool PRE, bool DY32>
void rn_bwd(const ResidArgs& a, bool sample, int grid, hipStream_t st) {
#define RN_GO(P, S) hipLaunchKernelGGL((resid_norm_bwd_kernel<WPR, P, S, PRE, B32, DY32>), dim3(grid), dim3(WPR == 1 ? 256 : 64 * WPR), 0, st, a)
    if (a.post_w) { if (sample) RN_GO(true, true); else RN_GO(true, false); }
    else { if (sample) RN_GO(false, true); else RN_GO(false, false); }
#undef RN_GO
}
// (the operands' types are part of the kernel: chosen at run time they kept the next row's loads from being issued together, 274 -> 399 us at
// 65792 x 1024)
template <int WPR>
void rn_bwd(const ResidArgs& a, bool sample, int grid, hipStream_t st) {
    if (!a.pre_w) { if (a.branch_f32) rn_bwd<WPR, true, false, false>(a, sample, grid, st); else rn_bwd<WPR, false, false, false>(a, sample, grid, st); }
    else if (a.dy_f32) { if (a.branch_f32) rn_bwd<WPR, true, true, true>(a, sample, grid, st); else rn_bwd<WPR, false, true, true>(a, sample, grid, st); }
    else { if (a.branch_f32) rn_bwd<WPR, true, true, false>(a, sample, grid, st); else rn_bwd<WPR, false, true, false>(a, sample, grid, st); }
}

int rn_check(const mrg_resid_norm_desc* d, const char* who) {
    MRG_REQUIRE(d != nullptr, MRG_ERR_ARG, "%s: null descriptor", who);
    MRG_REQUIRE(d->D >= 4 && d->D <= 4096 && d->D % 4 == 0, MRG_ERR_SHAPE, "%s: D = %d (a multiple of 4 up to 4096)", who, d->D);
    MRG_REQUIRE(d->samples >= 0 && d->rows_per_sample >= 0 && (long)d->samples * d->rows_per_sample <= 0x7ffffff0l, MRG_ERR_SHAPE, "%s: bad row counts", who);
    MRG_REQUIRE(d->norm == MRG_NORM_LAYER || d->norm == MRG_NORM_RMS, MRG_ERR_ARG, "%s: unknown norm %d", who, d->norm);
    MRG_REQUIRE(d->branch_dtype == MRG_DT_BF16 || d->branch_dtype == MRG_DT_F32, MRG_ERR_ARG, "%s: branch dtype", who);
    MRG_REQUIRE(d->y_dtype == MRG_DT_BF16 || d->y_dtype == MRG_DT_F32, MRG_ERR_ARG, "%s: y dtype", who);
    MRG_REQUIRE(d->gate_rows == 0 || d->gate_rows == 1 || d->gate_rows == d->samples, MRG_ERR_SHAPE, "%s: %d gate rows for %d samples", who, d->gate_rows, d->samples);
    MRG_REQUIRE((d->gate_rows == 0) == (d->gate == nullptr) || d->samples == 0, MRG_ERR_ARG, "%s: gate and gate_rows disagree", who);
    MRG_REQUIRE((d->post_b == nullptr || d->post_w) && (d->pre_b == nullptr || d->pre_w), MRG_ERR_ARG, "%s: a norm's bias without its weight", who);
    const void* vec[] = {d->x, d->branch, d->gate, d->post_w, d->post_b, d->pre_w, d->pre_b, d->x_new, d->y, d->dx_new, d->dy, d->dx, d->dbranch};
    for (const void* p : vec) MRG_REQUIRE((uintptr_t)p % 16 == 0, MRG_ERR_ARG, "%s: operands must be 16-byte aligned", who);
    return MRG_OK;
}

ResidArgs rn_args(const mrg_resid_norm_desc* d) {
    ResidArgs a = {};
    a.x = d->x; a.branch = d->branch; a.gate = d->gate; a.gate_stride = d->gate_rows > 1 ? d->D : 0; a.alpha = d->alpha;
    a.post_w = d->post_w; a.post_b = d->post_b; a.pre_w = d->pre_w; a.pre_b = d->pre_b;
    a.x_new = d->x_new; a.y = d->y; a.y_f32 = d->y_dtype == MRG_DT_F32; a.stats = d->stats;
    a.M = d->samples * d->rows_per_sample; a.L = d->rows_per_sample; a.D = d->D; a.layer = d->norm == MRG_NORM_LAYER; a.eps = d->eps;
    a.dx_new = d->dx_new; a.dy = d->dy; a.dy_f32 = a.y_f32; a.branch_f32 = d->branch_dtype == MRG_DT_F32; a.dx = d->dx; a.dbranch = d->dbranch;
    return a;
}

// rows that share a gate: a gate per sample keeps the samples apart, otherwise the whole batch is one
void rn_scope(const mrg_resid_norm_desc* d, int& scopes, int& rows, int& parts) {
    const bool sample = d->gate_rows > 1;
    scopes = sample ? d->samples : 1;
    rows = sample ? d->rows_per_sample : d->samples * d->rows_per_sample;
    parts = rn_parts(scopes, rows, d->D);
}

}  // namespace

extern "C" int mrg_resid_norm_fwd(const mrg_resid_norm_desc* d, hipStream_t stream) {
    const int rc = rn_check(d, "mrg_resid_norm_fwd");
    if (rc) return rc;
    ResidArgs a = rn_args(d);
    if (a.M == 0) return MRG_OK;
    MRG_REQUIRE(d->x && d->branch && d->x_new && (!d->pre_w || d->y) && ((!d->pre_w && !d->post_w) || d->stats), MRG_ERR_ARG, "mrg_resid_norm_fwd: null pointer");
    const bool wide = d->D > 1024, f = d->branch_dtype == MRG_DT_F32;
    const int nv = wide ? (d->D + 1023) / 1024 : (d->D + 255) / 256;
    // a launch has less than 2^32 threads along a dimension
    const long blocks = wide ? a.M : ((long)a.M + 3) / 4, across = blocks < (1l << 24) ? blocks : 1l << 23;
    const dim3 grid((unsigned)across, (unsigned)((blocks + across - 1) / across));
#define RN_F(NV, WPR) do { if (f) hipLaunchKernelGGL((resid_norm_fwd_kernel<NV, WPR, true>), grid, dim3(256), 0, stream, a); \
                           else hipLaunchKernelGGL((resid_norm_fwd_kernel<NV, WPR, false>), grid, dim3(256), 0, stream, a); } while (0)
    if (wide) { if (nv == 2) RN_F(2, 4); else if (nv == 3) RN_F(3, 4); else RN_F(4, 4); }
    else { if (nv == 1) RN_F(1, 1); else if (nv == 2) RN_F(2, 1); else if (nv == 3) RN_F(3, 1); else RN_F(4, 1); }
#undef RN_F
    return mrg_check_launch("mrg_resid_norm_fwd");
}

extern "C" long mrg_resid_norm_ws_floats(const mrg_resid_norm_desc* d) {
    if (rn_check(d, "mrg_resid_norm_ws_floats")) return -1;
    int scopes, rows, parts;
    rn_scope(d, scopes, rows, parts);
    const long units = (long)scopes * parts;
    return units ? ((long)rn_grid(units, d->D) * 4 + units) * d->D : 0;
}

extern "C" int mrg_resid_norm_bwd(const mrg_resid_norm_desc* d, hipStream_t stream) {
    const int rc = rn_check(d, "mrg_resid_norm_bwd");
    if (rc) return rc;
    ResidArgs a = rn_args(d);
    MRG_REQUIRE(a.M == 0 || (d->dx_new && d->branch && d->dx && d->dbranch && d->ws && (!d->pre_w || (d->dy && d->x_new)) && ((!d->pre_w && !d->post_w) || d->stats)),
                MRG_ERR_ARG, "mrg_resid_norm_bwd: null pointer");
    MRG_REQUIRE((!d->pre_w || d->d_pre_w) && (!d->pre_b || d->d_pre_b) && (!d->post_w || d->d_post_w) && (!d->post_b || d->d_post_b) && (d->gate_rows == 0 || d->d_gate),
                MRG_ERR_ARG, "mrg_resid_norm_bwd: missing gradient destination");
    const void* vec[] = {d->ws, d->d_pre_w, d->d_pre_b, d->d_post_w, d->d_post_b, d->d_gate};
    for (const void* p : vec) MRG_REQUIRE((uintptr_t)p % 16 == 0, MRG_ERR_ARG, "mrg_resid_norm_bwd: gradients must be 16-byte aligned");
    const bool sample = d->gate_rows > 1;
    int scopes, rows, parts;
    rn_scope(d, scopes, rows, parts);
    a.L = rows; a.parts = parts; a.units = a.M ? scopes * parts : 0;
    const int grid = a.M ? rn_grid(a.units, d->D) : 0;
    const bool gated = d->gate_rows > 0;
    a.part = d->ws; a.gpart = gated ? d->ws + (long)grid * 4 * d->D : nullptr;
    if (a.M) {
        switch (rn_waves(d->D)) {
            case 1: rn_bwd<1>(a, sample, grid, stream); break;
            case 2: rn_bwd<2>(a, sample, grid, stream); break;
            case 3: rn_bwd<3>(a, sample, grid, stream); break;
            case 4: rn_bwd<4>(a, sample, grid, stream); break;
            case 8: rn_bwd<8>(a, sample, grid, stream); break;
            default: rn_bwd<16>(a, sample, grid, stream);
        }
    }
    // the partial rows' sums (no rows at all: every gradient is zero)
    SumArgs s = {};
    int njobs = 0;
    const long ps = 4l * d->D;
    float* dst[4] = {d->pre_w ? d->d_pre_w : nullptr, d->pre_b ? d->d_pre_b : nullptr, d->post_w ? d->d_post_w : nullptr, d->post_b ? d->d_post_b : nullptr};
    for (int q = 0; q < 4; ++q) if (dst[q]) s.job[njobs++] = SumJob{a.part + (long)q * d->D, dst[q], grid, ps};
    s.gsrc = a.gpart; s.gdst = d->d_gate; s.D = d->D;
    s.parts = a.M == 0 ? 0 : (sample ? parts : grid);
    const int gates = gated ? (sample ? d->samples : 1) : 0;
    s.njobs = njobs; s.jobs = njobs + gates;
    const int across = s.jobs < (1 << 23) ? s.jobs : 1 << 23;
    if (s.jobs) hipLaunchKernelGGL(resid_norm_sum_kernel, dim3(across, (d->D / 4 + 7) / 8), dim3(256), 0, stream, s);
    return mrg_check_launch("mrg_resid_norm_bwd");
}
