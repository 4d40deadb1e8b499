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
// Measured, 16 384 x 4 096 bf16: forward 112 us (106 at a large copy's 5.05 TB/s), backward 166 us and 6 for the sums (160).
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

// V elements by one load: 16 bytes, two 16-bit elements, or one element
template <typename T, int V> struct alignas(V * sizeof(T)) Few { T v[V]; };
template <typename T, int V> __device__ inline void get(const void* base, long long at, float* o) {
    const Few<T, V> q = *(const Few<T, V>*)((const T*)base + at);
#pragma unroll
    for (int i = 0; i < V; i++) o[i] = (float)q.v[i];
}
template <typename T, int V> __device__ inline void put(void* base, long long at, const float* v) {
    Few<T, V> q;
#pragma unroll
    for (int i = 0; i < V; i++) q.v[i] = (T)v[i];
    *(Few<T, V>*)((T*)base + at) = q;
}

// One row in registers as it lies in memory.
template <typename T, int V, int N> struct RawRow {
    Few<T, V> e[N];
    template <int LANES> __device__ inline void load(const void* base, long long at, int lane, int c) {
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int col = (n * LANES + lane) * V;
            if (col < c) e[n] = *(const Few<T, V>*)((const T*)base + at + col);
            else {
#pragma unroll
                for (int i = 0; i < V; i++) e[n].v[i] = (T)0.f;
            }
        }
    }
};

// two sums over the LANES lanes that share a row, the same values in each.  More than a wave: through LDS, `buf` used in turn so that one
// barrier an exchange is enough (a wave can be at most one exchange ahead of another).
template <int LANES> struct RowSum {
    float2* lds;
    int turn = 0;
    __device__ void operator()(float& a, float& b) {
        if constexpr (LANES <= 16) {
            a = LANES == 4 ? sum4(a) : sum16(a);
            b = LANES == 4 ? sum4(b) : sum16(b);
            return;
        }
        a = wave_sum(a);
        b = wave_sum(b);
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

// A workgroup goes through rows, ROWS at a time, LANES lanes a row.  With up to 16 columns a lane (8 in a workgroup of 1 024, which has half the
// registers), what multiplies and adds to a column (scale * gate * w1, scale * gate * b1, w2, b2) stays in registers until the gate changes, and
// the next row's loads go out before this one's sums are waited for: 74 400 x 902 fp16 457 -> 119 us (106 at the rate of a copy), where the six
// vectors were read again for each row in accesses as narrow as the rows'.
template <typename T, int V, int N, int LANES>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void block_norm_fwd(const NormFwd a) {
    constexpr int THREADS = LANES < 256 ? 256 : LANES, ROWS = THREADS / LANES;
    constexpr bool KEEP = N * V <= (LANES == 1024 ? 8 : 16);
    __shared__ float2 lds[2 * (THREADS / 64)];
    RowSum<LANES> row_sum{lds};
    const int lane = threadIdx.x % LANES;
    const float inv_c = 1.f / (float)a.c;
    const long long step = (long long)gridDim.x * ROWS;
    long long r = (long long)blockIdx.x * ROWS + threadIdx.x / LANES, gate_end = 0, gate_row = 0;
    float k1[KEEP ? N : 1][V], k0[KEEP ? N : 1][V], k3[KEEP ? N : 1][V], k2[KEEP ? N : 1][V];
    auto fill = [&](float* o, float v) {
#pragma unroll
        for (int i = 0; i < V; i++) o[i] = v;
    };
    auto times = [&](float* o, const void* p, long long at) {
        if (!p) return;
        float q[V];
        get<T, V>(p, at, q);
#pragma unroll
        for (int i = 0; i < V; i++) o[i] *= q[i];
    };
    // u = k1 yhat + k0, scale and gate included
    auto factors = [&](int col, float* w, float* b) {
        float g[V];
        fill(g, 1);
        fill(w, 1);
        fill(b, 0);
        if (col >= a.c) return;
        times(g, a.gate, gate_row + col);
        times(g, a.scale, col);
        times(w, a.w1, col);
        if (a.b1) get<T, V>(a.b1, col, b);
#pragma unroll
        for (int i = 0; i < V; i++) { w[i] *= g[i]; b[i] *= g[i]; }
    };
    auto factors2 = [&](int col, float* w, float* b) {
        fill(w, 1);
        fill(b, 0);
        if (col >= a.c) return;
        times(w, a.w2, col);
        if (a.b2) get<T, V>(a.b2, col, b);
    };
    if constexpr (KEEP) {
        if (a.z) {
#pragma unroll
            for (int n = 0; n < N; n++) factors2((n * LANES + lane) * V, k3[n], k2[n]);
        }
    }
    RawRow<T, V, N> y, x;
    auto load = [&](long long r) {
        if (a.y) y.template load<LANES>(a.y, r * a.ys, lane, a.c);
        x.template load<LANES>(a.x, r * a.xs, lane, a.c);
    };
    if (KEEP && r < a.rows) load(r);
    for (; r < a.rows; r += step) {
        if constexpr (!KEEP) load(r);
        const RawRow<T, V, N> yc = y, xc = x;
        if (KEEP && r + step < a.rows) load(r + step);
        if (a.y && r >= gate_end) {
            if (a.gate) {
                const long long g = r / a.per_gate;
                gate_row = g * a.c;
                gate_end = (g + 1) * a.per_gate;
            } else gate_end = a.rows;
            if constexpr (KEEP) {
#pragma unroll
                for (int n = 0; n < N; n++) factors((n * LANES + lane) * V, k1[n], k0[n]);
            }
        }
        float v[N][V];
        float mean_y = 0, rstd_y = 0, s = 0, none = 0;
        if (a.y) {
#pragma unroll
            for (int n = 0; n < N; n++)
#pragma unroll
                for (int i = 0; i < V; i++) { v[n][i] = (float)yc.e[n].v[i]; s += v[n][i]; }
            if (a.layer) { row_sum(s, none); mean_y = s * inv_c; }
            s = 0;
#pragma unroll
            for (int n = 0; n < N; n++) {
                if ((n * LANES + lane) * V < a.c) {
#pragma unroll
                    for (int i = 0; i < V; i++) { v[n][i] -= mean_y; s += v[n][i] * v[n][i]; }
                }
            }
            row_sum(s, none);
            rstd_y = 1.f / sqrtf(s * inv_c + a.eps);
        }
        s = 0;
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int col = (n * LANES + lane) * V;
            float h[V];
#pragma unroll
            for (int i = 0; i < V; i++) h[i] = (float)xc.e[n].v[i];
            if (a.y && col < a.c) {
                float w[V], b[V];
                if constexpr (!KEEP) factors(col, w, b);
#pragma unroll
                for (int i = 0; i < V; i++) h[i] += v[n][i] * rstd_y * (KEEP ? k1[KEEP ? n : 0][i] : w[i]) + (KEEP ? k0[KEEP ? n : 0][i] : b[i]);
            }
            if (col < a.c) put<T, V>(a.h, r * a.hs + col, h);
#pragma unroll
            for (int i = 0; i < V; i++) { v[n][i] = h[i]; s += h[i]; }
        }
        float mean_h = 0, rstd_h = 0;
        if (a.z) {
            if (a.layer) { row_sum(s, none); mean_h = s * inv_c; }
            s = 0;
#pragma unroll
            for (int n = 0; n < N; n++) {
                if ((n * LANES + lane) * V < a.c) {
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
                    float w[V], b[V];
                    if constexpr (!KEEP) factors2(col, w, b);
#pragma unroll
                    for (int i = 0; i < V; i++) v[n][i] = v[n][i] * rstd_h * (KEEP ? k3[KEEP ? n : 0][i] : w[i]) + (KEEP ? k2[KEEP ? n : 0][i] : b[i]);
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
    long long span;                  // rows of a part (whole gates: gates)
    long long parts_per_gate;        // > 0: a part lies inside one gate's rows; 0: a part is whole gates (their dgate is written at once)
    int c;
};

// A workgroup is a part: ROWS rows at a time, LANES lanes a row.  The vectors stay in registers (KEEP) and the next row's loads go out before this one's
// sums are waited for (AHEAD) where there are registers for it beside the four sums a column (a workgroup of 1 024 has half: 8 000 x 5 999 fp16 156 us with its
// six columns a lane kept, 224 read again; layer 164 and 250).  WHOLE: gates change within the part -- A and B are added up gate by gate; else the
// gate is one number a column and P = sum t yhat, T = sum t give A, B and Q at the end.
template <typename T, int V, int N, int LANES, bool LAYER, bool WHOLE>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void block_norm_bwd(const NormBwd a) {
    constexpr int THREADS = LANES < 256 ? 256 : LANES, ROWS = THREADS / LANES;
    constexpr bool AHEAD = !WHOLE && N * V * sizeof(T) <= 32 && N <= 8 && LANES <= 512, KEEP = !WHOLE && N * V <= (LANES <= 512 ? 16 : 6);
    __shared__ float2 lds[2 * (THREADS / 64)];
    __shared__ float sums[LANES < 256 ? THREADS * V * N : 1];
    RowSum<LANES> row_sum{lds};
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const float inv_c = 1.f / (float)a.c;
    const long long part = blockIdx.x;
    long long r0, r1, gate = 0, gates_left = 0;
    const int stride = WHOLE ? 1 : ROWS;
    if (WHOLE) {                     // gates sub, sub + ROWS, ... of the part's
        const long long g0 = part * a.span + sub, g1 = min((part + 1) * a.span, a.rows / a.per_gate);
        gate = g0;
        gates_left = g0 < g1 ? (g1 - g0 + ROWS - 1) / ROWS : 0;
        r0 = g0 * a.per_gate;
        r1 = r0 + (gates_left ? a.per_gate : 0);
    } else {
        gate = part / a.parts_per_gate;
        const long long k = part % a.parts_per_gate;
        r0 = gate * a.per_gate + min(k * a.span, a.per_gate) + sub;
        r1 = gate * a.per_gate + min((k + 1) * a.span, a.per_gate);
    }
    float P[N][V], Tt[LAYER ? N : 1][V], W[N][V], D[LAYER ? N : 1][V], A[WHOLE ? N : 1][V], B[WHOLE && LAYER ? N : 1][V];
    float k1[KEEP ? N : 1][V], k2[KEEP ? N : 1][V];
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int i = 0; i < V; i++) {
            P[n][i] = W[n][i] = 0;
            if constexpr (LAYER) Tt[n][i] = D[n][i] = 0;
            if constexpr (WHOLE) A[n][i] = 0;
            if constexpr (WHOLE && LAYER) B[n][i] = 0;
        }
    // scale * gate * post_weight, and pre_weight, of the lane's columns
    auto one = [&](float* o) {
#pragma unroll
        for (int i = 0; i < V; i++) o[i] = 1;
    };
    auto factor = [&](int n, int col, float* o, bool weight) {
        float q[V];
        one(o);
        if (col >= a.c) return;
        if (a.scale) get<T, V>(a.scale, col, o);
        if (a.gate) {
            get<T, V>(a.gate, gate * a.c + col, q);
#pragma unroll
            for (int i = 0; i < V; i++) o[i] *= q[i];
        }
        if (weight && a.w1) {
            get<T, V>(a.w1, col, q);
#pragma unroll
            for (int i = 0; i < V; i++) o[i] *= q[i];
        }
    };
    auto factor2 = [&](int col, float* o) {
        one(o);
        if (a.w2 && col < a.c) get<T, V>(a.w2, col, o);
    };
    if constexpr (KEEP) {
#pragma unroll
        for (int n = 0; n < N; n++) {
            factor(n, (n * LANES + lane) * V, k1[n], true);
            factor2((n * LANES + lane) * V, k2[n]);
        }
    }
    RawRow<T, V, N> dz, h, dh, y;
    float4 st = make_float4(0, 0, 0, 0);
    auto load = [&](long long r) {
        st = *(const float4*)(a.stats + r * 4);
        if (a.dz) {
            dz.template load<LANES>(a.dz, r * a.dzs, lane, a.c);
            h.template load<LANES>(a.h, r * a.hs, lane, a.c);
        }
        if (a.dh) dh.template load<LANES>(a.dh, r * a.dhs, lane, a.c);
        if (a.y) y.template load<LANES>(a.y, r * a.ys, lane, a.c);
    };
    // (rows a workgroup shares: every lane of it goes through the same rows, barriers included)
    for (;;) {
        if (AHEAD && r0 < r1) load(r0);
        for (long long r = r0; r < r1; r += stride) {
            RawRow<T, V, N> dzc, hc, dhc, yc;
            float4 s4;
            if constexpr (!AHEAD) load(r);
            dzc = dz; hc = h; dhc = dh; yc = y; s4 = st;
            if (AHEAD && r + stride < r1) load(r + stride);
            float t[N][V], e[N][V], s1 = 0, s2 = 0;
            if (a.dz) {
#pragma unroll
                for (int n = 0; n < N; n++) {
                    float w[V];
                    if constexpr (!KEEP) factor2((n * LANES + lane) * V, w);
                    const bool in = (n * LANES + lane) * V < a.c;
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        const float d = (float)dzc.e[n].v[i];
                        e[n][i] = in ? ((float)hc.e[n].v[i] - s4.z) * s4.w : 0.f;
                        W[n][i] += d * e[n][i];
                        if constexpr (LAYER) D[n][i] += d;
                        t[n][i] = d * (KEEP ? k2[KEEP ? n : 0][i] : w[i]);
                        s1 += t[n][i];
                        s2 += t[n][i] * e[n][i];
                    }
                }
                row_sum(s1, s2);
                s1 = LAYER ? s1 * inv_c : 0.f;
                s2 *= inv_c;
            }
#pragma unroll
            for (int n = 0; n < N; n++)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    t[n][i] = a.dz ? s4.w * (t[n][i] - s1 - e[n][i] * s2) : 0.f;
                    if (a.dh) t[n][i] += (float)dhc.e[n].v[i];
                }
            if (a.dx) {
#pragma unroll
                for (int n = 0; n < N; n++) {
                    const int col = (n * LANES + lane) * V;
                    if (col < a.c) put<T, V>(a.dx, r * a.dxs + col, t[n]);
                }
            }
            if (!a.y) continue;
            s1 = s2 = 0;
#pragma unroll
            for (int n = 0; n < N; n++) {
                float w[V];
                const int col = (n * LANES + lane) * V;
                if constexpr (!KEEP) factor(n, col, w, true);
                const bool in = col < a.c;
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float ti = in ? t[n][i] : 0.f, yh = in ? ((float)yc.e[n].v[i] - s4.x) * s4.y : 0.f;
                    P[n][i] += ti * yh;
                    if constexpr (LAYER) Tt[n][i] += ti;
                    const float d = ti * (KEEP ? k1[KEEP ? n : 0][i] : w[i]);
                    t[n][i] = d; e[n][i] = yh;
                    s1 += d; s2 += d * yh;
                }
            }
            if (!a.dy) continue;
            row_sum(s1, s2);
            s1 = LAYER ? s1 * inv_c : 0.f;
            s2 *= inv_c;
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int col = (n * LANES + lane) * V;
                if (col < a.c) {
#pragma unroll
                    for (int i = 0; i < V; i++) t[n][i] = s4.y * (t[n][i] - s1 - e[n][i] * s2);
                    put<T, V>(a.dy, r * a.dys + col, t[n]);
                }
            }
        }
        if constexpr (!WHOLE) break;
        else {
            if (gates_left <= 0) break;
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int col = (n * LANES + lane) * V;
                if (col < a.c) {
                    float g[V], s[V], w[V], b[V];
                    one(g); one(s); one(w);
#pragma unroll
                    for (int i = 0; i < V; i++) b[i] = 0;
                    if (a.gate) get<T, V>(a.gate, gate * a.c + col, g);
                    if (a.scale) get<T, V>(a.scale, col, s);
                    if (a.w1) get<T, V>(a.w1, col, w);
                    if (a.b1) get<T, V>(a.b1, col, b);
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        const float tt = LAYER ? Tt[LAYER ? n : 0][i] : 0.f;
                        A[n][i] += g[i] * P[n][i];
                        if constexpr (LAYER) { B[n][i] += g[i] * tt; Tt[n][i] = 0; }
                        s[i] *= w[i] * P[n][i] + b[i] * tt;
                        P[n][i] = 0;
                    }
                    if (a.dgate) put<T, V>(a.dgate, gate * a.c + col, s);
                }
            }
            gates_left--;
            gate += ROWS;
            r0 = gate * a.per_gate;
            r1 = r0 + (gates_left > 0 ? a.per_gate : 0);
        }
    }
    if (!a.part) return;
    // the workgroup's sums: where several rows were handled side by side, added through LDS
    auto write = [&](int which, auto value) {
        float* o = a.part + (part * 5 + which) * a.c;
        if constexpr (LANES >= 256) {
#pragma unroll
            for (int n = 0; n < N; n++)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const int col = (n * LANES + lane) * V + i;
                    if (col < a.c) o[col] = value(n, i, col);
                }
        } else {
            __syncthreads();
#pragma unroll
            for (int n = 0; n < N; n++)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const int col = (n * LANES + lane) * V + i;
                    sums[sub * (LANES * N * V) + col] = col < a.c ? value(n, i, col) : 0.f;
                }
            __syncthreads();
            for (int col = threadIdx.x; col < a.c; col += THREADS) {
                float s = 0;
#pragma unroll
                for (int k = 0; k < ROWS; k++) s += sums[k * (LANES * N * V) + col];
                o[col] = s;
            }
        }
    };
    auto vec = [&](const void* p, long long at, float other) { return p ? (float)((const T*)p)[at] : other; };
    if (a.y) {
        if constexpr (WHOLE) {
            write(0, [&](int n, int i, int) { return A[n][i]; });
            if constexpr (LAYER) write(1, [&](int n, int i, int) { return B[n][i]; });
        } else {
            write(0, [&](int n, int i, int col) { return P[n][i] * vec(a.gate, gate * a.c + col, 1.f); });
            if constexpr (LAYER) write(1, [&](int n, int i, int col) { return Tt[n][i] * vec(a.gate, gate * a.c + col, 1.f); });
            if (a.dgate) write(4, [&](int n, int i, int col) { return P[n][i] * vec(a.w1, col, 1.f) + (LAYER ? Tt[LAYER ? n : 0][i] * vec(a.b1, col, 0.f) : 0.f); });
        }
    }
    if (a.dz) {
        write(2, [&](int n, int i, int) { return W[n][i]; });
        if constexpr (LAYER) write(3, [&](int n, int i, int) { return D[n][i]; });
    }
}

// The vectors' gradients from the parts, added in a fixed order by 32 columns x 32 lanes of parts (64 x 16 where
// rows are long: whole lines).  Job 0: of post_*, 1: of pre_*, 2 + j: dgate's row j.
struct NormEnd {
    const float* part;
    const void *scale, *w1, *b1;
    void *dgate, *dscale, *dw1, *db1, *dw2, *db2;
    long long parts, parts_per_gate;
    int c, col_blocks, layer, post, pre;
};
template <typename T, int COLS>
__global__ __launch_bounds__(1024) void block_norm_end(const NormEnd a) {
    constexpr int LANES = 1024 / COLS;
    __shared__ float lds[2][LANES][COLS];
    const int cb = blockIdx.x % a.col_blocks;
    const long long job = blockIdx.x / a.col_blocks;
    const int k = threadIdx.x / COLS, lane = threadIdx.x % COLS, col = cb * COLS + lane;
    if ((job == 0 && !a.post) || (job == 1 && !a.pre)) return;
    const long long p0 = job > 1 ? (job - 2) * a.parts_per_gate : 0, p1 = job > 1 ? p0 + a.parts_per_gate : a.parts;
    const int first = job > 1 ? 4 : (int)job * 2;
    const bool two = job < 2 && a.layer;
    float s0 = 0, s1 = 0;
    if (col < a.c) {
        const float* q = a.part + first * (long long)a.c + col;
        const long long step = 5 * (long long)a.c;
        if (two) {
#pragma unroll 8
            for (long long p = p0 + k; p < p1; p += LANES) { s0 += q[p * step]; s1 += q[p * step + a.c]; }
        } else {
#pragma unroll 8
            for (long long p = p0 + k; p < p1; p += LANES) s0 += q[p * step];
        }
    }
    lds[0][k][lane] = s0;
    lds[1][k][lane] = s1;
    __syncthreads();
    if (k || col >= a.c) return;
    s0 = s1 = 0;
#pragma unroll
    for (int i = 0; i < LANES; i++) { s0 += lds[0][i][lane]; s1 += lds[1][i][lane]; }
    const float sc = a.scale ? (float)((const T*)a.scale)[col] : 1.f;
    if (job > 1) {
        ((T*)a.dgate)[(job - 2) * a.c + col] = (T)(s0 * sc);
        return;
    }
    if (job == 1) {
        if (a.dw2) ((T*)a.dw2)[col] = (T)s0;
        if (a.db2) ((T*)a.db2)[col] = (T)s1;
        return;
    }
    const float w = a.w1 ? (float)((const T*)a.w1)[col] : 1.f, b = a.b1 ? (float)((const T*)a.b1)[col] : 0.f;
    if (a.dscale) ((T*)a.dscale)[col] = (T)(w * s0 + b * s1);
    if (a.dw1) ((T*)a.dw1)[col] = (T)(sc * s0);
    if (a.db1) ((T*)a.db1)[col] = (T)(sc * s1);
}

template <typename T> static void (*end_kernel(int cols))(NormEnd) { return cols == 32 ? block_norm_end<T, 32> : block_norm_end<T, 64>; }

static_assert(sizeof(aipt_block_norm_args) == 152 && sizeof(aipt_block_norm_grad_args) == 224, "argument records (api.py packs them by field)");

// ---- which kernel: the fewest lanes that hold a row; 16-byte accesses where every row begins at 16 bytes, two 16-bit elements where at 4 (74 400 rows of
// 902 fp16: 111 us by twos; of 901 one by one: 166).  Up to 8 or 16 columns a lane, so that the vectors stay in registers: 4 lanes for 32 columns of 16
// bits rather than 16 (65 964 rows: 13 -> 7 us, backward 25 -> 15), 256 for 2 048 rather than 64 with 32 columns each (16 384 rows: 92 -> 55), 512 for
// 8 192 rather than 256 (8 192 rows: 237 -> 120), 256 for 999 fp16 by ones in the backward pass rather than 64 (20 000 rows: 187 -> 75).  One by one, six
// columns a lane up to 6 144 (8 000 x 5 999 fp16: 125 us and backward 156, where eight and sixteen take 159 and 174; layer 151 and 164, 191 and 249), and in the
// backward pass 512 lanes of sixteen up to 8 192, which 1 024 lanes have no registers for (6 000 x 7 999 fp16: 163 us, 882).
// Whole gates (g*): a lane holds two sums a column more, and so few kernels serve them: half the shapes.  All of the others' would take 16 384 x 2 048 bf16 of 2 048
// gates from 297 to 167 us and 8 192 x 8 192 from 829 to 302, but 200 000 x 101 from 262 to 382 and 200 000 x 32 from 194 to 226.
struct NormShape { int v, n, lanes; };
template <int S> static NormShape norm_shape(int c, int v, const int (&shapes)[S][2]) {
    for (auto& s : shapes) if (s[0] * s[1] * v >= c) return {v, s[1], s[0]};
    return {0, 0, 0};
}
static NormShape fwd_shape(int es, int c, int v) {
    static const int w8[][2] = {{4, 1}, {16, 1}, {16, 2}, {64, 1}, {64, 2}, {256, 1}, {256, 2}, {512, 2}, {1024, 2}},
                     w4[][2] = {{4, 1}, {16, 1}, {16, 2}, {64, 1}, {64, 2}, {64, 4}, {256, 2}, {256, 4}, {1024, 2}, {1024, 4}},
                     twos[][2] = {{16, 2}, {16, 4}, {64, 4}, {64, 8}, {256, 4}, {256, 8}, {512, 8}, {1024, 8}},
                     ones[][2] = {{16, 2}, {16, 4}, {16, 8}, {64, 4}, {64, 8}, {256, 4}, {256, 8}, {512, 8}, {1024, 6}, {1024, 8}, {1024, 16}};
    return v == 1 ? norm_shape(c, 1, ones) : v == 8 ? norm_shape(c, 8, w8) : v == 4 ? norm_shape(c, 4, w4) : norm_shape(c, 2, twos);
}
static NormShape bwd_shape(int es, int c, int v, bool whole) {
    static const int w8[][2] = {{4, 1}, {16, 1}, {16, 2}, {64, 2}, {256, 1}, {256, 2}, {512, 2}, {1024, 2}}, w4[][2] = {{4, 1}, {16, 1}, {16, 2}, {64, 2}, {256, 1}, {256, 2}, {256, 4}, {512, 4}, {1024, 4}},
                     twos[][2] = {{16, 2}, {16, 4}, {64, 4}, {256, 2}, {256, 4}, {256, 8}, {512, 8}, {1024, 8}}, ones[][2] = {{16, 2}, {16, 4}, {16, 8}, {64, 8}, {256, 4}, {256, 8}, {512, 8}, {1024, 6}, {512, 16}, {1024, 16}};
    static const int g8[][2] = {{16, 1}, {64, 2}, {256, 2}, {1024, 2}}, g4[][2] = {{16, 1}, {64, 2}, {256, 2}, {1024, 4}}, gones[][2] = {{16, 4}, {64, 8}, {256, 8}, {1024, 8}, {1024, 16}};
    if (whole) return v != 16 / es ? norm_shape(c, 1, gones) : es == 2 ? norm_shape(c, 8, g8) : norm_shape(c, 4, g4);
    return v == 1 ? norm_shape(c, 1, ones) : v != 16 / es ? norm_shape(c, 2, twos) : es == 2 ? norm_shape(c, 8, w8) : norm_shape(c, 4, w4);
}

template <typename T> static void (*fwd_kernel(NormShape s))(NormFwd) {
    constexpr int V = 16 / sizeof(T);
#define AIPT_FWD(VV, NN, LL) if (s.v == VV && s.n == NN && s.lanes == LL) return block_norm_fwd<T, VV, NN, LL>;
    AIPT_FWD(V, 1, 4) AIPT_FWD(V, 1, 16) AIPT_FWD(V, 2, 16) AIPT_FWD(V, 1, 64) AIPT_FWD(V, 2, 64) AIPT_FWD(V, 2, 256) AIPT_FWD(V, 2, 1024)
    if constexpr (V == 4) { AIPT_FWD(V, 4, 64) AIPT_FWD(V, 4, 256) AIPT_FWD(V, 4, 1024) }
    else { AIPT_FWD(V, 1, 256) AIPT_FWD(V, 2, 512) AIPT_FWD(2, 2, 16) AIPT_FWD(2, 4, 16) AIPT_FWD(2, 4, 64) AIPT_FWD(2, 8, 64) AIPT_FWD(2, 4, 256) AIPT_FWD(2, 8, 256) AIPT_FWD(2, 8, 512) AIPT_FWD(2, 8, 1024) }
    AIPT_FWD(1, 2, 16) AIPT_FWD(1, 4, 16) AIPT_FWD(1, 8, 16) AIPT_FWD(1, 4, 64) AIPT_FWD(1, 8, 64) AIPT_FWD(1, 4, 256) AIPT_FWD(1, 8, 256) AIPT_FWD(1, 8, 512) AIPT_FWD(1, 6, 1024) AIPT_FWD(1, 8, 1024)
    AIPT_FWD(1, 16, 1024)
    return nullptr;
#undef AIPT_FWD
}
template <typename T, bool LAYER> static void (*bwd_kernel(NormShape s, bool whole))(NormBwd) {
    constexpr int V = 16 / sizeof(T);
#define AIPT_BWD(VV, NN, LL, GG) if (s.v == VV && s.n == NN && s.lanes == LL && whole == GG) return block_norm_bwd<T, VV, NN, LL, LAYER, GG>;
    AIPT_BWD(V, 1, 4, false) AIPT_BWD(V, 1, 16, false) AIPT_BWD(V, 2, 16, false) AIPT_BWD(V, 2, 64, false) AIPT_BWD(V, 1, 256, false) AIPT_BWD(V, 2, 256, false)
    if constexpr (V == 8) {
        AIPT_BWD(V, 2, 512, false) AIPT_BWD(V, 2, 1024, false) AIPT_BWD(V, 2, 1024, true)
        AIPT_BWD(2, 2, 16, false) AIPT_BWD(2, 4, 16, false) AIPT_BWD(2, 4, 64, false) AIPT_BWD(2, 2, 256, false) AIPT_BWD(2, 4, 256, false) AIPT_BWD(2, 8, 256, false) AIPT_BWD(2, 8, 512, false) AIPT_BWD(2, 8, 1024, false)
    } else { AIPT_BWD(V, 4, 256, false) AIPT_BWD(V, 4, 512, false) AIPT_BWD(V, 4, 1024, false) AIPT_BWD(V, 4, 1024, true) }
    AIPT_BWD(V, 1, 16, true) AIPT_BWD(V, 2, 64, true) AIPT_BWD(V, 2, 256, true)
    AIPT_BWD(1, 2, 16, false) AIPT_BWD(1, 4, 16, false) AIPT_BWD(1, 8, 16, false) AIPT_BWD(1, 8, 64, false) AIPT_BWD(1, 4, 256, false) AIPT_BWD(1, 8, 256, false) AIPT_BWD(1, 8, 512, false) AIPT_BWD(1, 6, 1024, false) AIPT_BWD(1, 16, 512, false)
    AIPT_BWD(1, 16, 1024, false) AIPT_BWD(1, 4, 16, true) AIPT_BWD(1, 8, 64, true) AIPT_BWD(1, 8, 256, true) AIPT_BWD(1, 8, 1024, true)
    AIPT_BWD(1, 16, 1024, true)
    return nullptr;
#undef AIPT_BWD
}

// Parts of the backward pass (a workgroup each): two a CU, one where a lane's columns fill its registers or the workgroup is larger (100 000 x 512 bf16
// layer 142 us with 512 parts, 171 with 768, 158 with 1 024; 16 384 x 4 096 bf16 rms 173 with 256, 182 with 512), none shorter than 4 rows for each
// row handled at a time.  Gates fewer than that are split into parts; more, and a part takes whole gates.
struct NormParts { long long parts, span, per_gate_parts; };
static bool norm_whole(long long groups) { return groups >= 512; }
static NormParts norm_parts(long long rows, long long groups, NormShape s) {
    const long long want = s.lanes < 256 || (s.lanes == 256 && s.n * s.v <= 8) ? 512 : 256, at_once = s.lanes < 256 ? 256 / s.lanes : 1;
    const long long per = std::max(1ll, rows / groups);
    NormParts p;
    if (norm_whole(groups)) {
        p.span = std::max(at_once, (groups + want - 1) / want);
        p.parts = (groups + p.span - 1) / p.span;
        p.per_gate_parts = 0;
    } else {
        long long k = std::max(1ll, std::min(want / groups, per / (4 * at_once)));
        p.span = (per + k - 1) / k;
        k = (per + p.span - 1) / p.span;
        p.parts = k * groups;
        p.per_gate_parts = k;
    }
    return p;
}

}  // namespace aipt

using aipt::fail;

// how many elements may move together: 16 bytes' worth, two of 16 bits, or one.  `strides`: 0 for what is not there.
static int norm_unit(int es, int c, long long rows, std::initializer_list<const void*> ptrs, std::initializer_list<long long> strides) {
    uintptr_t all = 0;
    for (const void* p : ptrs) all |= (uintptr_t)p;
    long long lines = c;
    if (rows > 1) for (long long s : strides) lines |= s;
    for (int v : {16 / es, 2}) if (v * es <= 16 && (es == 2 || v == 4) && !(all & (v * es - 1)) && !(lines & (v - 1))) return v;
    return 1;
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
    const int v = norm_unit(es, a->c, a->rows, {a->x, a->y, a->h, a->z, a->gate, a->scale, a->post_weight, a->post_bias, a->pre_weight, a->pre_bias},
                            {a->x_stride, a->h_stride, a->y ? a->y_stride : 0, a->z ? a->z_stride : 0});
    const aipt::NormShape s = aipt::fwd_shape(es, a->c, v);
    const aipt::NormFwd f = {a->x, a->y, a->gate, a->scale, a->post_weight, a->post_bias, a->pre_weight, a->pre_bias, a->h, a->z, a->stats,
                             a->rows, a->rows / (a->gate ? a->groups : 1), a->x_stride, a->y_stride, a->h_stride, a->z_stride, a->c, a->kind == AIPT_NORM_LAYER, a->eps};
    const int threads = std::max(256, s.lanes), per = threads / s.lanes;
    const long long want = (a->rows + per - 1) / per;
    // 1 024 threads a CU, 512 where a lane holds more than 8 columns (its registers leave no more): 16 384 x 2 048 bf16 78 us with 512, 55 with
    // 1 024 and 58 with 2 048; 74 400 x 902 fp16 146, 111, 136 us with 256, 512 and 1 024.
    const size_t blocks = (size_t)std::min(want, (s.n * s.v <= 8 ? 1024ll : 512ll) * 256 / threads);
    auto* k = a->type == AIPT_TYPE_F32 ? aipt::fwd_kernel<float>(s) : a->type == AIPT_TYPE_BF16 ? aipt::fwd_kernel<aipt::bf16>(s) : aipt::fwd_kernel<aipt::f16>(s);
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
    const long long groups = norm_gated(a) ? a->groups : 1;
    size_t most = 0;
    const int es = aipt::type_bytes(a->type);
    for (int v : {1, 2, 16 / es}) {
        if (v == 2 && es == 4) continue;
        const aipt::NormShape s = aipt::bwd_shape(es, a->c, v, aipt::norm_whole(groups));
        const aipt::NormParts p = aipt::norm_parts(std::max(1ll, a->rows), groups, s);
        most = std::max(most, (size_t)p.parts * 5 * a->c * sizeof(float));
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
    const int v = norm_unit(es, a->c, a->rows, {a->dh, a->dz, a->y, a->dz ? a->h : nullptr, a->gate, a->scale, a->post_weight, a->post_bias, a->pre_weight, a->dx, a->dy, a->dgate},
                            {strides[0], strides[1], strides[2], strides[3], a->dx ? a->dx_stride : 0, a->dy ? a->dy_stride : 0});
    const long long groups = norm_gated(a) ? a->groups : 1;
    const bool whole = aipt::norm_whole(groups);
    const aipt::NormShape s = aipt::bwd_shape(es, a->c, v, whole);
    const int threads = std::max(256, s.lanes);
    const aipt::NormParts p = aipt::norm_parts(a->rows, groups, s);
    const size_t blocks = (size_t)p.parts;
    const bool part = sums || (a->dgate && p.per_gate_parts);
    const size_t need = part ? blocks * 5 * a->c * sizeof(float) : 0;
    if (need && (!d_workspace || workspace_bytes < need)) return fail(ctx, AIPT_E_INVALID, "%s: workspace of %zu bytes, %zu are wanted", me, workspace_bytes, need);
    const aipt::NormBwd b = {a->dh, a->dz, a->y, a->h, a->gate, a->scale, a->post_weight, a->post_bias, a->pre_weight, a->stats, a->dx, a->dy, a->dgate,
                             part ? (float*)d_workspace : nullptr, a->rows, std::max(1ll, a->rows / groups), a->dh_stride, a->dz_stride, a->y_stride, a->h_stride, a->dx_stride, a->dy_stride,
                             p.span, p.per_gate_parts, a->c};
    const bool layer = a->kind == AIPT_NORM_LAYER;
    auto pick = [&](auto t) { return layer ? aipt::bwd_kernel<decltype(t), true>(s, whole) : aipt::bwd_kernel<decltype(t), false>(s, whole); };
    auto* k = a->type == AIPT_TYPE_F32 ? pick(0.f) : a->type == AIPT_TYPE_BF16 ? pick((aipt::bf16)0.f) : pick((aipt::f16)0.f);
    if (!aipt::grid_fits(blocks, threads)) return fail(ctx, AIPT_E_INVALID, "%s: %lld rows of %lld groups are too many", me, a->rows, a->groups);
    AIPT_NEED_CTX(ctx);
    aipt::DeviceScope dev(ctx->device);
    AIPT_HIP(ctx, dev.err);
    AIPT_HIP(ctx, aipt::launch(k, blocks, threads, 0, ctx->stream, b));
    if (part) {
        const int cols = a->c <= 1024 ? 32 : 64, cb = (a->c + cols - 1) / cols;
        const bool gates = a->dgate && p.per_gate_parts;
        const aipt::NormEnd e = {(const float*)d_workspace, a->scale, a->post_weight, a->post_bias, a->dgate, a->dscale, a->dpost_weight, a->dpost_bias, a->dpre_weight, a->dpre_bias,
                                 p.parts, p.per_gate_parts, a->c, cb, layer, a->dscale || a->dpost_weight || a->dpost_bias, a->dpre_weight || a->dpre_bias};
        const size_t jobs = 2 + (gates ? (size_t)a->groups : 0);
        auto* ke = a->type == AIPT_TYPE_F32 ? aipt::end_kernel<float>(cols) : a->type == AIPT_TYPE_BF16 ? aipt::end_kernel<aipt::bf16>(cols) : aipt::end_kernel<aipt::f16>(cols);
        AIPT_HIP(ctx, aipt::launch(ke, jobs * cb, 1024, 0, ctx->stream, e));
    }
    return AIPT_OK;
}

}  // extern "C"
