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
// Bound: HBM.  Forward reads 4 + 2 and writes 4 + 2 bytes an element (fp32 residual, bf16 branch and y), backward reads 12 and writes 6.
// A row is read once into registers (a wave per row up to 1024 columns, four waves beyond), all statistics in fp32: the mean first, then the
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
    const float* dx_new; const void* dy; int dy_f32; float* dx; void* dbranch;
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

// sum over the lanes of a row: its wave, or its four waves through `box` (two alternating sets of slots; every wave of the workgroup calls it
// the same number of times)
template <int WPR>
struct RowSum {
    float (*box)[2][4]; int turn = 0, wave;
    __device__ __forceinline__ float2 operator()(float a, float b) {
        a = wave_sum(a); b = wave_sum(b);
        if (WPR == 1) return make_float2(a, b);
        float (&slot)[2][4] = box[turn];
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) { slot[0][wave] = a; slot[1][wave] = b; }
        __syncthreads();
        return make_float2((slot[0][0] + slot[0][1]) + (slot[0][2] + slot[0][3]), (slot[1][0] + slot[1][1]) + (slot[1][2] + slot[1][3]));
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
    __shared__ float box[2][2][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = WPR == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
    if (WPR == 1 && row >= a.M) return;
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

// SAMPLE: a gate per sample -- the sums A and T are closed at the end of every unit (a part of one sample's rows) into gpart and into the
// workgroup's own dw_post / db_post; otherwise there is one gate (or none) and they are closed once
template <int NV, int WPR, bool BR32, bool POST, bool SAMPLE>
__global__ __launch_bounds__(256) void resid_norm_bwd_kernel(const ResidArgs a) {
    __shared__ float box[2][2][4];
    __shared__ __attribute__((aligned(16))) float buf[WPR == 1 ? 4 * NV * 256 : 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    RowSum<WPR> sum{box, 0, wave};
    const int D = a.D, nv = D >> 2, c0 = WPR == 1 ? lane : threadIdx.x, step = 64 * WPR;
    const float invD = 1.f / (float)D;
    bool ok[NV];
    float4 pre_w[NV], post_w[NV], g[NV], sw[NV], sb[NV], A[NV], T[NV], GA[NV], GT[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = c0 + step * j;
        ok[j] = c < nv;
        pre_w[j] = (ok[j] && a.pre_w) ? reinterpret_cast<const float4*>(a.pre_w)[c] : zero4();
        post_w[j] = (ok[j] && POST) ? reinterpret_cast<const float4*>(a.post_w)[c] : zero4();
        g[j] = make_float4(1.f, 1.f, 1.f, 1.f);
        if (!SAMPLE && ok[j] && a.gate) g[j] = reinterpret_cast<const float4*>(a.gate)[c];
        sw[j] = sb[j] = A[j] = T[j] = GA[j] = GT[j] = zero4();
    }
    // one column sum of the workgroup: its waves' registers meet in LDS (a wave per row) or are whole already (a row over four waves)
    auto flush = [&](const float4 (&v)[NV], float* out) {
        if (WPR == 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NV; ++j) if (ok[j]) reinterpret_cast<float4*>(buf + wave * NV * 256)[c0 + step * j] = v[j];
            __syncthreads();
            for (int c = threadIdx.x; c < D; c += 256) out[c] = (buf[c] + buf[NV * 256 + c]) + (buf[2 * NV * 256 + c] + buf[3 * NV * 256 + c]);
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j) if (ok[j]) reinterpret_cast<float4*>(out)[c0 + step * j] = v[j];
        }
    };
    // end of the rows that share a gate: dgate = w_post A + b_post T, and g A, g T towards dw_post, db_post
    auto close = [&](int slot) {
        if (a.gpart) {
            float4 dg[NV];
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                dg[j] = POST ? A[j] * post_w[j] : A[j];
                if (POST && ok[j] && a.post_b) dg[j] = dg[j] + T[j] * reinterpret_cast<const float4*>(a.post_b)[c0 + step * j];
            }
            flush(dg, a.gpart + (long)slot * D);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            GA[j] = GA[j] + A[j] * g[j]; GT[j] = GT[j] + T[j] * g[j];
            if (SAMPLE) A[j] = T[j] = zero4();
        }
    };
    const int u0 = (int)((long)blockIdx.x * a.units / gridDim.x), u1 = (int)((long)(blockIdx.x + 1) * a.units / gridDim.x);
    for (int u = u0; u < u1; ++u) {
        const int smp = u / a.parts, part = u - smp * a.parts;
        const int lo = smp * a.L + (int)((long)part * a.L / a.parts), hi = smp * a.L + (int)((long)(part + 1) * a.L / a.parts);
        if (SAMPLE) {
#pragma unroll
            for (int j = 0; j < NV; ++j) if (ok[j]) g[j] = reinterpret_cast<const float4*>(a.gate + (long)smp * a.gate_stride)[c0 + step * j];
        }
        for (int row = lo + (WPR == 1 ? wave : 0); row < hi; row += (WPR == 1 ? 4 : 1)) {
            float4 t[NV], w[NV], xh[NV], b[NV];
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = c0 + step * j;
                t[j] = w[j] = xh[j] = b[j] = zero4();
                if (ok[j]) {
                    t[j] = rn_load(a.dx_new, row, D, c, true);
                    b[j] = rn_load(a.branch, row, D, c, BR32);
                    if (a.pre_w) { w[j] = rn_load(a.dy, row, D, c, a.dy_f32); xh[j] = rn_load(a.x_new, row, D, c, true); }
                }
            }
            if (a.pre_w) {
                const float mu = a.stats[2l * a.M + row], rs = a.stats[3l * a.M + row];
                float s1 = 0.f, s2 = 0.f;
#pragma unroll
                for (int j = 0; j < NV; ++j) if (ok[j]) {
                    xh[j] = scale4(shift4(xh[j], mu), rs);
                    sw[j] = sw[j] + w[j] * xh[j];
                    sb[j] = sb[j] + w[j];
                    w[j] = w[j] * pre_w[j];
                    s1 += sum4(w[j]); s2 += dot4(w[j], xh[j]);
                }
                const float2 m = sum(s1, s2);
                const float m1 = a.layer ? m.x * invD : 0.f, m2 = m.y * invD;
#pragma unroll
                for (int j = 0; j < NV; ++j) if (ok[j]) t[j] = fma4(fma4(xh[j], -m2, shift4(w[j], m1)), rs, t[j]);
            }
            float rs = 1.f;
            if (POST) {
                const float mu = a.stats[row];
                rs = a.stats[(long)a.M + row];
#pragma unroll
                for (int j = 0; j < NV; ++j) if (ok[j]) b[j] = scale4(shift4(b[j], mu), rs);
            }
            float s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int j = 0; j < NV; ++j) if (ok[j]) {
                rn_store(a.dx, row, D, c0 + step * j, true, scale4(t[j], a.alpha));
                A[j] = A[j] + t[j] * b[j];
                if (POST) T[j] = T[j] + t[j];
                t[j] = t[j] * g[j];
                if (POST) { t[j] = t[j] * post_w[j]; s1 += sum4(t[j]); s2 += dot4(t[j], b[j]); }
            }
            if (POST) {
                const float2 m = sum(s1, s2);
                const float m1 = a.layer ? m.x * invD : 0.f, m2 = m.y * invD;
#pragma unroll
                for (int j = 0; j < NV; ++j) if (ok[j]) t[j] = scale4(fma4(b[j], -m2, shift4(t[j], m1)), rs);
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) if (ok[j]) rn_store(a.dbranch, row, D, c0 + step * j, BR32, t[j]);
        }
        if (SAMPLE) close(u);
    }
    if (!SAMPLE) close(blockIdx.x);
    float* out = a.part + (long)blockIdx.x * 4 * D;
    if (a.pre_w) { flush(sw, out); if (a.pre_b) flush(sb, out + D); }
    if (POST) { flush(GA, out + 2 * D); if (a.post_b) flush(GT, out + 3 * D); }
}

// column sums of the partial rows: job j (blockIdx.x) adds `n` rows that lie `stride` floats apart.  32 columns and 32 rows at a time; the
// order of the additions is fixed by the sizes alone
struct SumJob { const float* src; float* dst; int n; long stride; };
struct SumArgs { SumJob job[4]; const float* gsrc; float* gdst; int parts, D; };
__global__ __launch_bounds__(256) void resid_norm_sum_kernel(const SumArgs a, int njobs) {
    __shared__ __attribute__((aligned(16))) float4 box[32][8];
    const int cl = threadIdx.x & 7, rl = threadIdx.x >> 3;
    const int c = blockIdx.y * 8 + cl;
    SumJob job;
    if ((int)blockIdx.x < njobs) job = a.job[blockIdx.x];
    else {
        const long s = (long)blockIdx.x - njobs;                  // one sample's gate: its parts are consecutive rows
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
    if (rl == 0 && c * 4 < a.D) reinterpret_cast<float4*>(job.dst)[c] = box[0][cl];
}

// units of the backward launch: the rows that share a gate, cut into `parts` so that about two workgroups per CU have work, but no part
// below 16 rows (four per wave) where a gate has that many
constexpr int RN_GRID = 512;
int rn_parts(int samples, int L) {
    int parts = (RN_GRID + samples - 1) / samples;
    const int most = (L + 15) / 16;
    return parts < 1 ? 1 : (parts > most ? (most < 1 ? 1 : most) : parts);
}
int rn_grid(long units) { return (int)(units < RN_GRID ? units : RN_GRID); }

template <int NV, int WPR, bool BR32>
void rn_bwd(const ResidArgs& a, bool post, bool sample, int grid, hipStream_t st) {
#define RN_GO(P, S) hipLaunchKernelGGL((resid_norm_bwd_kernel<NV, WPR, BR32, P, S>), dim3(grid), dim3(256), 0, st, a)
    if (post) { if (sample) RN_GO(true, true); else RN_GO(true, false); }
    else { if (sample) RN_GO(false, true); else RN_GO(false, false); }
#undef RN_GO
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
    a.dx_new = d->dx_new; a.dy = d->dy; a.dy_f32 = a.y_f32; a.dx = d->dx; a.dbranch = d->dbranch;
    return a;
}

// rows that share a gate: a gate per sample keeps the samples apart, otherwise the whole batch is one
void rn_scope(const mrg_resid_norm_desc* d, int& scopes, int& rows, int& parts) {
    const bool sample = d->gate_rows > 1;
    scopes = sample ? d->samples : 1;
    rows = sample ? d->rows_per_sample : d->samples * d->rows_per_sample;
    parts = rn_parts(scopes, rows);
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
    const dim3 grid(wide ? a.M : (a.M + 3) / 4);
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
    return ((long)rn_grid(units) * 4 + units) * d->D;
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
    const int grid = a.M ? rn_grid(a.units) : 0;
    const bool gated = d->gate_rows > 0;
    a.part = d->ws; a.gpart = gated ? d->ws + (long)grid * 4 * d->D : nullptr;
    if (a.M) {
        const bool wide = d->D > 1024, f = d->branch_dtype == MRG_DT_F32, post = d->post_w != nullptr;
        const int nv = wide ? (d->D + 1023) / 1024 : (d->D + 255) / 256;
#define RN_B(NV, WPR) do { if (f) rn_bwd<NV, WPR, true>(a, post, sample, grid, stream); else rn_bwd<NV, WPR, false>(a, post, sample, grid, stream); } while (0)
        if (wide) { if (nv == 2) RN_B(2, 4); else if (nv == 3) RN_B(3, 4); else RN_B(4, 4); }
        else { if (nv == 1) RN_B(1, 1); else if (nv == 2) RN_B(2, 1); else if (nv == 3) RN_B(3, 1); else RN_B(4, 1); }
#undef RN_B
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
    if (njobs + gates) hipLaunchKernelGGL(resid_norm_sum_kernel, dim3(njobs + gates, (d->D / 4 + 7) / 8), dim3(256), 0, stream, s, njobs);
    return mrg_check_launch("mrg_resid_norm_bwd");
}
