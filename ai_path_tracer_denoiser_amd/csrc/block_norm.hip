// block_norm.hip -- the norms around a residual block with its gate and residual scale, forward and backward (aipt_block_norm*).
//
//     u = norm(y) * w1 + b1;   h = x + s * g * u;   z = norm(h) * w2 + b2
//
// Forward: y and x in, h and z out, nothing else can be saved: memory bounds it.  A row stays in the registers of the lanes that
// share it (a wave, or a workgroup for long rows), so both norms' statistics are two-pass -- the mean, then the squares of
// what is left of it -- without a second read.
//
// Backward, with t = dh + norm'(dz * w2) the gradient of the residual stream (dx = t), d = t s g w1, dy = norm'(d):
//     norm'(d) = rstd (d - mean(d) [layer only] - vhat mean(d * vhat))
// dh, dz, y, h in, dx and dy out.  The gradients of the vectors are sums over rows; with
//     A = sum g t yhat,  B = sum g t,  Q = sum_(rows of a gate) t (w1 yhat + b1),  W = sum dz hhat,  V = sum dz
// they are  dw1 = s A,  db1 = s B,  ds = w1 A + b1 B,  dgate = s Q,  dw2 = W,  db2 = V: four (five) sums a column, which each
// workgroup keeps in registers over the rows it handles and writes once; a second, small launch adds those in a fixed order.
#include "layer_ops.h"

namespace aipt {

struct NormFwd {
    const void *x, *y, *gate, *scale, *w1, *b1, *w2, *b2;
    void *h, *z;
    float* stats;
    long long rows, per_gate, xs, ys, hs, zs;
    int c, layer;
    float eps;
};

// V elements from p: one 16-byte load, or one element
template <typename T, int V> __device__ inline void get(const void* base, long long at, float* o) {
    if constexpr (V == 1) o[0] = (float)((const T*)base)[at];
    else {
        const Chunk<T> q = *(const Chunk<T>*)((const T*)base + at);
#pragma unroll
        for (int i = 0; i < V; i++) o[i] = (float)q.v[i];
    }
}
template <typename T, int V> __device__ inline void put(void* base, long long at, const float* v) {
    if constexpr (V == 1) ((T*)base)[at] = (T)v[0];
    else {
        Chunk<T> q;
#pragma unroll
        for (int i = 0; i < V; i++) q.v[i] = (T)v[i];
        *(Chunk<T>*)((T*)base + at) = q;
    }
}

// two sums over the LANES lanes that share a row, the same values in each.  More than a wave: through LDS, `buf` used in turn so that one
// barrier an exchange is enough (a wave can be at most one exchange ahead of another).
template <int LANES> struct RowSum {
    float2* lds;
    int turn = 0;
    __device__ void operator()(float& a, float& b) {
#pragma unroll
        for (int o = 32; o; o >>= 1) { a += __shfl_xor(a, o); b += __shfl_xor(b, o); }
        if constexpr (LANES > 64) {
            constexpr int W = LANES / 64;
            float2* s = lds + turn * W;
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = make_float2(a, b);
            __syncthreads();
            a = b = 0;
#pragma unroll
            for (int i = 0; i < W; i++) { a += s[i].x; b += s[i].y; }
        }
    }
};

template <typename T, int V, int N, int LANES>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void block_norm_fwd(const NormFwd a) {
    constexpr int THREADS = LANES < 256 ? 256 : LANES, ROWS = THREADS / LANES;
    __shared__ float2 lds[2 * (THREADS / 64)];
    RowSum<LANES> row_sum{lds};
    const int lane = threadIdx.x % LANES;
    const float inv_c = 1.f / (float)a.c;
    for (long long r = (long long)blockIdx.x * ROWS + threadIdx.x / LANES; r < a.rows; r += (long long)gridDim.x * ROWS) {
        float v[N][V];
        float mean_y = 0, rstd_y = 0;
        if (a.y) {
            float s = 0, none = 0;
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int col = (n * LANES + lane) * V;
                if (col < a.c) get<T, V>(a.y, r * a.ys + col, v[n]);
                else {
#pragma unroll
                    for (int i = 0; i < V; i++) v[n][i] = 0;
                }
#pragma unroll
                for (int i = 0; i < V; i++) s += v[n][i];
            }
            if (a.layer) { row_sum(s, none); mean_y = s * inv_c; }
            s = 0;
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int col = (n * LANES + lane) * V;
                if (col < a.c) {
#pragma unroll
                    for (int i = 0; i < V; i++) { v[n][i] -= mean_y; s += v[n][i] * v[n][i]; }
                }
            }
            row_sum(s, none);
            rstd_y = 1.f / sqrtf(s * inv_c + a.eps);
        }
        const long long gate_row = a.gate ? r / a.per_gate * a.c : 0;
        float s = 0, none = 0;
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int col = (n * LANES + lane) * V;
            if (col < a.c) {
                float h[V], q[V];
                get<T, V>(a.x, r * a.xs + col, h);
                if (a.y) {
#pragma unroll
                    for (int i = 0; i < V; i++) v[n][i] *= rstd_y;
                    if (a.w1) { get<T, V>(a.w1, col, q);
#pragma unroll
                        for (int i = 0; i < V; i++) v[n][i] *= q[i]; }
                    if (a.b1) { get<T, V>(a.b1, col, q);
#pragma unroll
                        for (int i = 0; i < V; i++) v[n][i] += q[i]; }
                    if (a.gate) { get<T, V>(a.gate, gate_row + col, q);
#pragma unroll
                        for (int i = 0; i < V; i++) v[n][i] *= q[i]; }
                    if (a.scale) { get<T, V>(a.scale, col, q);
#pragma unroll
                        for (int i = 0; i < V; i++) v[n][i] *= q[i]; }
#pragma unroll
                    for (int i = 0; i < V; i++) h[i] += v[n][i];
                }
                put<T, V>(a.h, r * a.hs + col, h);
#pragma unroll
                for (int i = 0; i < V; i++) { v[n][i] = h[i]; s += h[i]; }
            }
        }
        float mean_h = 0, rstd_h = 0;
        if (a.z) {
            if (a.layer) { row_sum(s, none); mean_h = s * inv_c; }
            s = 0;
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int col = (n * LANES + lane) * V;
                if (col < a.c) {
#pragma unroll
                    for (int i = 0; i < V; i++) { v[n][i] -= mean_h; s += v[n][i] * v[n][i]; }
                }
            }
            row_sum(s, none);
            rstd_h = 1.f / sqrtf(s * inv_c + a.eps);
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int col = (n * LANES + lane) * V;
                if (col < a.c) {
                    float q[V];
#pragma unroll
                    for (int i = 0; i < V; i++) v[n][i] *= rstd_h;
                    if (a.w2) { get<T, V>(a.w2, col, q);
#pragma unroll
                        for (int i = 0; i < V; i++) v[n][i] *= q[i]; }
                    if (a.b2) { get<T, V>(a.b2, col, q);
#pragma unroll
                        for (int i = 0; i < V; i++) v[n][i] += q[i]; }
                    put<T, V>(a.z, r * a.zs + col, v[n]);
                }
            }
        }
        if (a.stats && lane == 0) *(float4*)(a.stats + r * 4) = make_float4(mean_y, rstd_y, mean_h, rstd_h);
    }
}

struct NormBwd {
    const void *dh, *dz, *y, *h, *gate, *scale, *w1, *b1, *w2;
    const float* stats;
    void *dx, *dy, *dgate;
    float* part;                     // [parts][5][c]: A, B, W, V, Q
    long long rows, per_gate, dhs, dzs, ys, hs, dxs, dys;
    long long span;                  // rows of a part
    long long parts_per_gate;        // > 0: a part lies inside one gate's rows; 0: a part is whole gates (their dgate is written at once)
    int c, layer, sums;              // sums: whether A, B, W, V are wanted (else dgate alone, or none)
};

template <typename T, int V, int N, int LANES>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void block_norm_bwd(const NormBwd a) {
    constexpr int THREADS = LANES < 256 ? 256 : LANES, ROWS = THREADS / LANES;
    __shared__ float2 lds[2 * (THREADS / 64)];
    RowSum<LANES> row_sum{lds};
    const int lane = threadIdx.x % LANES;
    const float inv_c = 1.f / (float)a.c;
    // a part is what LANES lanes handle: rows [r0, r1), one after the other
    const long long part = (long long)blockIdx.x * ROWS + threadIdx.x / LANES;
    long long r0, r1;
    if (a.parts_per_gate) {
        const long long gate = part / a.parts_per_gate, k = part % a.parts_per_gate;
        r0 = gate * a.per_gate + min(k * a.span, a.per_gate);
        r1 = gate * a.per_gate + min((k + 1) * a.span, a.per_gate);
        if (r0 > a.rows) r0 = a.rows;
        if (r1 > a.rows) r1 = a.rows;
    } else {
        r0 = min(part * a.span, a.rows);
        r1 = min((part + 1) * a.span, a.rows);
    }
    float A[N][V], B[N][V], W[N][V], D[N][V], Q[N][V];
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int i = 0; i < V; i++) A[n][i] = B[n][i] = W[n][i] = D[n][i] = Q[n][i] = 0;
    long long gate_left = 0;         // rows to go of the present gate (whole gates only)
    for (long long r = r0; r < r1; r++) {
        const float4 st = *(const float4*)(a.stats + r * 4);
        float t[N][V], e[N][V];
        float s1 = 0, s2 = 0;
        // t = dh + norm'(dz w2); e: hhat
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int col = (n * LANES + lane) * V;
#pragma unroll
            for (int i = 0; i < V; i++) t[n][i] = e[n][i] = 0;
            if (a.dz && col < a.c) {
                float d[V], w[V];
                get<T, V>(a.dz, r * a.dzs + col, d);
                get<T, V>(a.h, r * a.hs + col, e[n]);
#pragma unroll
                for (int i = 0; i < V; i++) {
                    e[n][i] = (e[n][i] - st.z) * st.w;
                    W[n][i] += d[i] * e[n][i];
                    D[n][i] += d[i];
                }
                if (a.w2) { get<T, V>(a.w2, col, w);
#pragma unroll
                    for (int i = 0; i < V; i++) d[i] *= w[i]; }
#pragma unroll
                for (int i = 0; i < V; i++) { t[n][i] = d[i]; s1 += d[i]; s2 += d[i] * e[n][i]; }
            }
        }
        if (a.dz) {
            row_sum(s1, s2);
            s1 = a.layer ? s1 * inv_c : 0.f;
            s2 *= inv_c;
#pragma unroll
            for (int n = 0; n < N; n++)
#pragma unroll
                for (int i = 0; i < V; i++) t[n][i] = st.w * (t[n][i] - s1 - e[n][i] * s2);
        }
        const long long gate_row = a.gate || a.dgate ? r / a.per_gate * a.c : 0;
        if (!a.parts_per_gate && a.dgate && gate_left == 0) gate_left = a.per_gate;
        s1 = s2 = 0;
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int col = (n * LANES + lane) * V;
            if (col < a.c) {
                float q[V];
                if (a.dh) { get<T, V>(a.dh, r * a.dhs + col, q);
#pragma unroll
                    for (int i = 0; i < V; i++) t[n][i] += q[i]; }
                if (a.dx) put<T, V>(a.dx, r * a.dxs + col, t[n]);
                if (a.y) {
                    float y[V], w[V], g[V], b[V], sc[V];
                    get<T, V>(a.y, r * a.ys + col, y);
#pragma unroll
                    for (int i = 0; i < V; i++) { y[i] = (y[i] - st.x) * st.y; w[i] = 1; g[i] = 1; b[i] = 0; sc[i] = 1; }
                    if (a.w1) get<T, V>(a.w1, col, w);
                    if (a.b1) get<T, V>(a.b1, col, b);
                    if (a.gate) get<T, V>(a.gate, gate_row + col, g);
                    if (a.scale) get<T, V>(a.scale, col, sc);
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        const float ti = t[n][i], gt = g[i] * ti;
                        A[n][i] += gt * y[i];
                        B[n][i] += gt;
                        Q[n][i] += ti * (w[i] * y[i] + b[i]);
                        const float d = gt * sc[i] * w[i];
                        t[n][i] = d; e[n][i] = y[i];
                        s1 += d; s2 += d * y[i];
                    }
                    if (!a.parts_per_gate && a.dgate && gate_left == 1) {
#pragma unroll
                        for (int i = 0; i < V; i++) { q[i] = Q[n][i] * sc[i]; Q[n][i] = 0; }
                        put<T, V>(a.dgate, gate_row + col, q);
                    }
                }
            }
        }
        gate_left--;
        if (a.y && a.dy) {
            row_sum(s1, s2);
            s1 = a.layer ? s1 * inv_c : 0.f;
            s2 *= inv_c;
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int col = (n * LANES + lane) * V;
                if (col < a.c) {
#pragma unroll
                    for (int i = 0; i < V; i++) t[n][i] = st.y * (t[n][i] - s1 - e[n][i] * s2);
                    put<T, V>(a.dy, r * a.dys + col, t[n]);
                }
            }
        }
    }
    if (a.part) {
        float* p = a.part + part * 5 * a.c;
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int col = (n * LANES + lane) * V + i;
                if (col < a.c) {
                    if (a.sums) { p[col] = A[n][i]; p[a.c + col] = B[n][i]; p[2 * a.c + col] = W[n][i]; p[3 * a.c + col] = D[n][i]; }
                    if (a.parts_per_gate) p[4 * a.c + col] = Q[n][i];
                }
            }
    }
}

// the vectors' gradients from the parts: blockIdx.y 0 adds A, B, W, V over all parts, blockIdx.y 1 + j adds Q over the parts of gate j.
// 64 columns x 4 lanes of parts, added in a fixed order.
struct NormEnd {
    const float* part;
    const void *scale, *w1, *b1;
    void *dgate, *dscale, *dw1, *db1, *dw2, *db2;
    long long parts, parts_per_gate;
    int c, col_blocks;
};
template <typename T>
__global__ __launch_bounds__(256) void block_norm_end(const NormEnd a) {
    __shared__ float lds[4][4][64];
    const int cb = blockIdx.x % a.col_blocks;
    const long long job = blockIdx.x / a.col_blocks;
    const int k = threadIdx.x >> 6, lane = threadIdx.x & 63, col = cb * 64 + lane;
    const bool in = col < a.c;
    const bool gates = job > 0;
    const long long p0 = gates ? (job - 1) * a.parts_per_gate : 0, p1 = gates ? p0 + a.parts_per_gate : a.parts;
    float s[4] = {};
    if (in)
        for (long long p = p0 + k; p < p1; p += 4) {
            const float* q = a.part + p * 5 * a.c + col;
            if (gates) s[0] += q[4 * (long long)a.c];
            else {
#pragma unroll
                for (int j = 0; j < 4; j++) s[j] += q[j * (long long)a.c];
            }
        }
#pragma unroll
    for (int j = 0; j < 4; j++) lds[k][j][lane] = s[j];
    __syncthreads();
    if (k || !in) return;
#pragma unroll
    for (int j = 0; j < 4; j++) s[j] = (lds[0][j][lane] + lds[1][j][lane]) + (lds[2][j][lane] + lds[3][j][lane]);
    const float sc = a.scale ? (float)((const T*)a.scale)[col] : 1.f;
    if (gates) {
        ((T*)a.dgate)[(job - 1) * a.c + col] = (T)(s[0] * sc);
        return;
    }
    const float w = a.w1 ? (float)((const T*)a.w1)[col] : 1.f, b = a.b1 ? (float)((const T*)a.b1)[col] : 0.f;
    if (a.dscale) ((T*)a.dscale)[col] = (T)(w * s[0] + b * s[1]);
    if (a.dw1) ((T*)a.dw1)[col] = (T)(sc * s[0]);
    if (a.db1) ((T*)a.db1)[col] = (T)(sc * s[1]);
    if (a.dw2) ((T*)a.dw2)[col] = (T)s[2];
    if (a.db2) ((T*)a.db2)[col] = (T)s[3];
}

static_assert(sizeof(aipt_block_norm_args) == 152 && sizeof(aipt_block_norm_grad_args) == 224, "argument records (api.py packs them by field)");

// ---- which kernel: the fewest lanes that hold a row, 16-byte accesses where every row begins at 16 bytes
struct NormShape { int v, n, lanes; };
template <int VEC> static NormShape norm_shape(int c, bool wide) {
    const int v = wide ? VEC : 1;
    static const struct { int n, lanes; } wides[] = {{1, 64}, {2, 64}, {4, 64}, {2, 256}, {4, 256}, {2, 1024}, {4, 1024}},
                                          ones[] = {{1, 64}, {2, 64}, {4, 64}, {8, 64}, {4, 256}, {8, 256}, {4, 1024}, {16, 1024}};
    if (wide) { for (auto& s : wides) if (s.n * s.lanes * v >= c) return {v, s.n, s.lanes}; }
    else { for (auto& s : ones) if (s.n * s.lanes >= c) return {v, s.n, s.lanes}; }
    return {0, 0, 0};
}

#define AIPT_NORM_KERNELS(NAME, ARGS)                                                              \
    template <typename T> static void (*NAME##_kernel(NormShape s))(ARGS) {                        \
        constexpr int V = 16 / sizeof(T);                                                          \
        if (s.v == V) {                                                                            \
            if (s.lanes == 64) return s.n == 1 ? NAME<T, V, 1, 64> : s.n == 2 ? NAME<T, V, 2, 64> : NAME<T, V, 4, 64>; \
            if (s.lanes == 256) return s.n == 2 ? NAME<T, V, 2, 256> : NAME<T, V, 4, 256>;         \
            return s.n == 2 ? NAME<T, V, 2, 1024> : NAME<T, V, 4, 1024>;                           \
        }                                                                                          \
        if (s.lanes == 64) return s.n == 1 ? NAME<T, 1, 1, 64> : s.n == 2 ? NAME<T, 1, 2, 64> : s.n == 4 ? NAME<T, 1, 4, 64> : NAME<T, 1, 8, 64>; \
        if (s.lanes == 256) return s.n == 4 ? NAME<T, 1, 4, 256> : NAME<T, 1, 8, 256>;             \
        return s.n == 4 ? NAME<T, 1, 4, 1024> : NAME<T, 1, 16, 1024>;                              \
    }
AIPT_NORM_KERNELS(block_norm_fwd, NormFwd)
AIPT_NORM_KERNELS(block_norm_bwd, NormBwd)

// parts of the backward pass: enough for every CU to hold several, none shorter than 4 rows where there are rows enough
struct NormParts { long long parts, span, per_gate_parts; };
static NormParts norm_parts(long long rows, long long groups, int lanes) {
    const long long want = lanes == 64 ? 4096 : lanes == 256 ? 1024 : 256;
    const long long per = std::max(1ll, rows / groups);
    NormParts p;
    if (groups >= want) {                                    // whole gates
        const long long gates = (groups + want - 1) / want;
        p.span = gates * per;
        p.parts = (groups + gates - 1) / gates;
        p.per_gate_parts = 0;
    } else {
        long long k = std::max(1ll, std::min(want / groups, (per + 3) / 4));
        p.span = (per + k - 1) / k;
        k = (per + p.span - 1) / p.span;
        p.parts = k * groups;
        p.per_gate_parts = k;
    }
    return p;
}

}  // namespace aipt

using aipt::fail;

static bool on16(std::initializer_list<const void*> ptrs) {
    uintptr_t all = 0;
    for (const void* p : ptrs) all |= (uintptr_t)p;
    return !(all & 15);
}

extern "C" {

int aipt_block_norm(aipt_ctx* ctx, const aipt_block_norm_args* a) {
    const char* me = "aipt_block_norm";
    if (!a) return fail(ctx, AIPT_E_INVALID, "%s: args is NULL", me);
    if (!aipt::type_ok(a->type)) return fail(ctx, AIPT_E_INVALID, "%s: type %d", me, a->type);
    if (a->kind != AIPT_NORM_RMS && a->kind != AIPT_NORM_LAYER) return fail(ctx, AIPT_E_INVALID, "%s: kind %d", me, a->kind);
    if (a->c < 1 || a->c > 16384) return fail(ctx, AIPT_E_INVALID, "%s: %d channels (1..16384)", me, a->c);
    if (a->rows < 0 || a->rows > (1ll << 40)) return fail(ctx, AIPT_E_INVALID, "%s: %lld rows", me, a->rows);
    if (a->groups < 1 || (a->gate && a->rows % a->groups)) return fail(ctx, AIPT_E_INVALID, "%s: %lld rows in %lld groups", me, a->rows, a->groups);
    if (!(a->eps >= 0.f)) return fail(ctx, AIPT_E_INVALID, "%s: eps %g", me, a->eps);
    if (a->kind == AIPT_NORM_RMS && (a->post_bias || a->pre_bias)) return fail(ctx, AIPT_E_INVALID, "%s: biases belong to AIPT_NORM_LAYER", me);
    const bool any = a->rows > 0;                            // (an empty tensor has no memory: with no rows NULL says nothing)
    if (any && !a->y && (a->gate || a->scale || a->post_weight || a->post_bias)) return fail(ctx, AIPT_E_INVALID, "%s: gate, scale and post_* belong to a block's output y", me);
    if (any && !a->z && (a->pre_weight || a->pre_bias)) return fail(ctx, AIPT_E_INVALID, "%s: pre_* belong to z", me);
    if (!a->rows) {
        AIPT_NEED_CTX(ctx);
        return AIPT_OK;
    }
    if (!a->x || !a->h) return fail(ctx, AIPT_E_INVALID, "%s: x or h is NULL", me);
    const int es = aipt::type_bytes(a->type);
    const long long lo = 0, hi = (1ll << 40);
    if (a->x_stride < lo || a->x_stride > hi || (a->y && (a->y_stride < lo || a->y_stride > hi)) || (a->rows > 1 && (a->h_stride < a->c || (a->z && a->z_stride < a->c))) || a->h_stride > hi || a->z_stride > hi)
        return fail(ctx, AIPT_E_INVALID, "%s: row strides %lld %lld %lld %lld of %d channels", me, a->x_stride, a->y_stride, a->h_stride, a->z_stride, a->c);
    const void* all[] = {a->x, a->y, a->h, a->z, a->gate, a->scale, a->post_weight, a->post_bias, a->pre_weight, a->pre_bias};
    for (const void* p : all) if ((uintptr_t)p & (es - 1)) return fail(ctx, AIPT_E_INVALID, "%s: misaligned pointer", me);
    if ((uintptr_t)a->stats & 15) return fail(ctx, AIPT_E_INVALID, "%s: stats is not 16-byte aligned", me);
    auto ext = [&](const void* p, long long lines, long long stride) { return aipt::Extent{(const char*)p, lines, (long long)a->c * es, stride * es}; };
    const aipt::Extent out[] = {ext(a->h, a->rows, a->h_stride), ext(a->z, a->rows, a->z_stride), {(const char*)a->stats, 1, a->rows * 16, 0}};
    const aipt::Extent in[] = {ext(a->x, a->rows, a->x_stride), ext(a->y, a->rows, a->y_stride), ext(a->gate, a->groups, a->c), ext(a->scale, 1, 0),
                               ext(a->post_weight, 1, 0), ext(a->post_bias, 1, 0), ext(a->pre_weight, 1, 0), ext(a->pre_bias, 1, 0)};
    for (int o = 0; o < 3; o++) {
        for (int i = 0; i < 8; i++)
            if (!(o == 0 && i == 0 && a->h == a->x && (a->h_stride == a->x_stride || a->rows == 1)) && aipt::overlap(out[o], in[i]))
                return fail(ctx, AIPT_E_INVALID, "%s: an output overlaps an input", me);
        for (int i = 0; i < o; i++) if (aipt::overlap(out[o], out[i])) return fail(ctx, AIPT_E_INVALID, "%s: outputs overlap", me);
    }
    const int vec = 16 / es;
    const bool wide = a->c % vec == 0 && on16({a->x, a->y, a->h, a->z, a->gate, a->scale, a->post_weight, a->post_bias, a->pre_weight, a->pre_bias}) &&
                      (a->rows == 1 || (!(a->x_stride % vec) && !(a->h_stride % vec) && !(a->y && a->y_stride % vec) && !(a->z && a->z_stride % vec)));
    const aipt::NormShape s = vec == 4 ? aipt::norm_shape<4>(a->c, wide) : aipt::norm_shape<8>(a->c, wide);
    const aipt::NormFwd f = {a->x, a->y, a->gate, a->scale, a->post_weight, a->post_bias, a->pre_weight, a->pre_bias, a->h, a->z, a->stats,
                             a->rows, a->rows / (a->gate ? a->groups : 1), a->x_stride, a->y_stride, a->h_stride, a->z_stride, a->c, a->kind == AIPT_NORM_LAYER, a->eps};
    const int threads = std::max(256, s.lanes), per = threads / s.lanes;
    const long long want = (a->rows + per - 1) / per;
    const size_t blocks = (size_t)std::min(want, 1ll << 20);
    auto* k = a->type == AIPT_TYPE_F32 ? aipt::block_norm_fwd_kernel<float>(s) : a->type == AIPT_TYPE_BF16 ? aipt::block_norm_fwd_kernel<aipt::bf16>(s) : aipt::block_norm_fwd_kernel<aipt::f16>(s);
    AIPT_NEED_CTX(ctx);
    aipt::DeviceScope dev(ctx->device);
    AIPT_HIP(ctx, dev.err);
    AIPT_HIP(ctx, aipt::launch(k, blocks, threads, 0, ctx->stream, f));
    return AIPT_OK;
}

// the checks that need no memory, the kernel and the parts: the same answer for the workspace and for the call.  The kernel's shape may differ
// between the two (a workspace is asked for without pointers), so the workspace holds the parts of either.
static int norm_grad_check(aipt_ctx* ctx, const char* me, const aipt_block_norm_grad_args* a) {
    if (!a) return fail(ctx, AIPT_E_INVALID, "%s: args is NULL", me);
    if (a->reserved) return fail(ctx, AIPT_E_INVALID, "%s: reserved is not 0", me);
    if (!aipt::type_ok(a->type)) return fail(ctx, AIPT_E_INVALID, "%s: type %d", me, a->type);
    if (a->kind != AIPT_NORM_RMS && a->kind != AIPT_NORM_LAYER) return fail(ctx, AIPT_E_INVALID, "%s: kind %d", me, a->kind);
    if (a->c < 1 || a->c > 16384) return fail(ctx, AIPT_E_INVALID, "%s: %d channels (1..16384)", me, a->c);
    if (a->rows < 0 || a->rows > (1ll << 40)) return fail(ctx, AIPT_E_INVALID, "%s: %lld rows", me, a->rows);
    if (a->groups < 1 || ((a->gate || a->dgate) && a->rows % a->groups)) return fail(ctx, AIPT_E_INVALID, "%s: %lld rows in %lld groups", me, a->rows, a->groups);
    if (a->kind == AIPT_NORM_RMS && (a->post_bias || a->dpost_bias || a->dpre_bias)) return fail(ctx, AIPT_E_INVALID, "%s: biases belong to AIPT_NORM_LAYER", me);
    return AIPT_OK;
}
static bool norm_gated(const aipt_block_norm_grad_args* a) { return a->gate || a->dgate; }

int aipt_block_norm_backward_workspace(aipt_ctx* ctx, const aipt_block_norm_grad_args* a, size_t* bytes) {
    const char* me = "aipt_block_norm_backward_workspace";
    if (!bytes) return fail(ctx, AIPT_E_INVALID, "%s: bytes is NULL", me);
    const int rc = norm_grad_check(ctx, me, a);
    if (rc) return rc;
    size_t most = 0;
    for (bool wide : {false, true}) {
        const aipt::NormShape s = aipt::type_bytes(a->type) == 4 ? aipt::norm_shape<4>(a->c, wide) : aipt::norm_shape<8>(a->c, wide);
        const int per = std::max(256, s.lanes) / s.lanes;
        const aipt::NormParts p = aipt::norm_parts(std::max(1ll, a->rows), norm_gated(a) ? a->groups : 1, s.lanes);
        most = std::max(most, (size_t)((p.parts + per - 1) / per * per) * 5 * a->c * sizeof(float));
    }
    *bytes = most;
    return AIPT_OK;
}

int aipt_block_norm_backward(aipt_ctx* ctx, const aipt_block_norm_grad_args* a, void* d_workspace, size_t workspace_bytes) {
    const char* me = "aipt_block_norm_backward";
    const int rc = norm_grad_check(ctx, me, a);
    if (rc) return rc;
    const bool any = a->rows > 0;
    if (any && !a->y && (a->gate || a->scale || a->post_weight || a->post_bias || a->dy || a->dgate || a->dscale || a->dpost_weight || a->dpost_bias))
        return fail(ctx, AIPT_E_INVALID, "%s: gate, scale, post_* and dy belong to a block's output y", me);
    if (any && !a->dz && (a->pre_weight || a->dpre_weight || a->dpre_bias)) return fail(ctx, AIPT_E_INVALID, "%s: pre_* belong to dz", me);
    if (any && !a->dh && !a->dz) return fail(ctx, AIPT_E_INVALID, "%s: neither dh nor dz", me);
    const int es = aipt::type_bytes(a->type);
    const bool sums = a->dscale || a->dpost_weight || a->dpost_bias || a->dpre_weight || a->dpre_bias;
    if (a->rows) {
        if (!a->stats) return fail(ctx, AIPT_E_INVALID, "%s: stats is NULL", me);
        if (a->dz && !a->h) return fail(ctx, AIPT_E_INVALID, "%s: dz without h", me);
    }
    const long long hi = (1ll << 40);
    const long long strides[] = {a->dh ? a->dh_stride : 0, a->dz ? a->dz_stride : 0, a->y ? a->y_stride : 0, a->dz ? a->h_stride : 0};
    for (long long s : strides) if (s < 0 || s > hi) return fail(ctx, AIPT_E_INVALID, "%s: row stride %lld", me, s);
    if (a->rows > 1 && ((a->dx && (a->dx_stride < a->c || a->dx_stride > hi)) || (a->dy && (a->dy_stride < a->c || a->dy_stride > hi))))
        return fail(ctx, AIPT_E_INVALID, "%s: row strides %lld, %lld of %d channels", me, a->dx_stride, a->dy_stride, a->c);
    const void* all[] = {a->dh, a->dz, a->y, a->h, a->gate, a->scale, a->post_weight, a->post_bias, a->pre_weight, a->dx, a->dy, a->dgate, a->dscale,
                         a->dpost_weight, a->dpost_bias, a->dpre_weight, a->dpre_bias};
    for (const void* p : all) if ((uintptr_t)p & (es - 1)) return fail(ctx, AIPT_E_INVALID, "%s: misaligned pointer", me);
    if (((uintptr_t)a->stats & 15) || ((uintptr_t)d_workspace & 15)) return fail(ctx, AIPT_E_INVALID, "%s: stats or workspace is not 16-byte aligned", me);
    auto ext = [&](const void* p, long long lines, long long stride) { return aipt::Extent{(const char*)p, lines, (long long)a->c * es, stride * es}; };
    const aipt::Extent out[] = {ext(a->dx, a->rows, a->dx_stride), ext(a->dy, a->rows, a->dy_stride), ext(a->dgate, a->groups, a->c), ext(a->dscale, 1, 0), ext(a->dpost_weight, 1, 0),
                                ext(a->dpost_bias, 1, 0), ext(a->dpre_weight, 1, 0), ext(a->dpre_bias, 1, 0), {(const char*)d_workspace, 1, (long long)workspace_bytes, 0}};
    const aipt::Extent in[] = {ext(a->dh, a->rows, a->dh_stride), ext(a->dz, a->rows, a->dz_stride), ext(a->y, a->rows, a->y_stride), ext(a->dz ? a->h : nullptr, a->rows, a->h_stride),
                               ext(a->gate, a->groups, a->c), ext(a->scale, 1, 0), ext(a->post_weight, 1, 0), ext(a->post_bias, 1, 0), ext(a->pre_weight, 1, 0),
                               {(const char*)a->stats, 1, a->rows * 16, 0}};
    for (int o = 0; o < 9; o++) {
        for (int i = 0; i < 10; i++)
            if (!(o == 0 && i == 0 && a->dx == a->dh && (a->dx_stride == a->dh_stride || a->rows == 1)) && aipt::overlap(out[o], in[i]))
                return fail(ctx, AIPT_E_INVALID, "%s: an output overlaps an input", me);
        for (int i = 0; i < o; i++) if (aipt::overlap(out[o], out[i])) return fail(ctx, AIPT_E_INVALID, "%s: outputs overlap", me);
    }
    if (!a->rows) {                                          // nothing to add up
        AIPT_NEED_CTX(ctx);
    aipt::DeviceScope dev(ctx->device);
        AIPT_HIP(ctx, dev.err);
        for (int o = 2; o < 8; o++) AIPT_HIP(ctx, aipt::zero_fill(ctx->stream, out[o].data, (size_t)(out[o].lines * out[o].len)));
        return AIPT_OK;
    }
    const int vec = 16 / es;
    bool wide = a->c % vec == 0 && on16({a->dh, a->dz, a->y, a->dz ? a->h : nullptr, a->gate, a->scale, a->post_weight, a->post_bias, a->pre_weight, a->dx, a->dy, a->dgate});
    if (a->rows > 1) {
        for (long long s : strides) wide = wide && !(s % vec);
        wide = wide && !(a->dx && a->dx_stride % vec) && !(a->dy && a->dy_stride % vec);
    }
    const aipt::NormShape s = vec == 4 ? aipt::norm_shape<4>(a->c, wide) : aipt::norm_shape<8>(a->c, wide);
    const int threads = std::max(256, s.lanes), per = threads / s.lanes;
    const long long groups = norm_gated(a) ? a->groups : 1;
    aipt::NormParts p = aipt::norm_parts(std::max(1ll, a->rows), groups, s.lanes);
    const size_t blocks = (size_t)((p.parts + per - 1) / per);
    const bool part = sums || (a->dgate && p.per_gate_parts);
    const size_t need = part ? blocks * per * 5 * a->c * sizeof(float) : 0;
    if (need && (!d_workspace || workspace_bytes < need)) return fail(ctx, AIPT_E_INVALID, "%s: workspace of %zu bytes, %zu are wanted", me, workspace_bytes, need);
    const aipt::NormBwd b = {a->dh, a->dz, a->y, a->h, a->gate, a->scale, a->post_weight, a->post_bias, a->pre_weight, a->stats, a->dx, a->dy, a->dgate,
                             part ? (float*)d_workspace : nullptr, a->rows, std::max(1ll, a->rows / groups), a->dh_stride, a->dz_stride, a->y_stride, a->h_stride, a->dx_stride, a->dy_stride,
                             p.span, p.per_gate_parts, a->c, a->kind == AIPT_NORM_LAYER, sums};
    auto* k = a->type == AIPT_TYPE_F32 ? aipt::block_norm_bwd_kernel<float>(s) : a->type == AIPT_TYPE_BF16 ? aipt::block_norm_bwd_kernel<aipt::bf16>(s) : aipt::block_norm_bwd_kernel<aipt::f16>(s);
    if (!aipt::grid_fits(blocks, threads)) return fail(ctx, AIPT_E_INVALID, "%s: %lld rows of %lld groups are too many", me, a->rows, a->groups);
    AIPT_NEED_CTX(ctx);
    aipt::DeviceScope dev(ctx->device);
    AIPT_HIP(ctx, dev.err);
    AIPT_HIP(ctx, aipt::launch(k, blocks, threads, 0, ctx->stream, b));
    if (part) {
        const int cb = (a->c + 63) / 64;
        const bool gates = a->dgate && p.per_gate_parts;
        const aipt::NormEnd e = {(const float*)d_workspace, a->scale, a->post_weight, a->post_bias, a->dgate, a->dscale, a->dpost_weight, a->dpost_bias, a->dpre_weight, a->dpre_bias,
                                 sums ? p.parts : 0, p.per_gate_parts, a->c, cb};
        const size_t jobs = 1 + (gates ? (size_t)a->groups : 0);
        auto* ke = a->type == AIPT_TYPE_F32 ? aipt::block_norm_end<float> : a->type == AIPT_TYPE_BF16 ? aipt::block_norm_end<aipt::bf16> : aipt::block_norm_end<aipt::f16>;
        AIPT_HIP(ctx, aipt::launch(ke, jobs * cb, 256, 0, ctx->stream, e));
    }
    return AIPT_OK;
}

}  // extern "C"
