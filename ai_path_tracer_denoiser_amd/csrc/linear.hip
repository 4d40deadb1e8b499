// linear.hip -- matrix product with bias, activation and residual in its epilogue, and its gradients (aipt_linear*).
//
//     C[i][j] = sum_k A[i][k] B[j][k],   then  z = C + bias,  y = act(z) + residual
//
// One kernel family serves the three products: y = x w^T (i = row, j = channel, k = channel in), dx = dz w and dw = dz^T x
// (the contraction runs over rows).  Operands come with either stride the unit one, so a tile is loaded along whichever axis is contiguous.
#include "layer_ops.h"

namespace aipt {

typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct GemmArgs {
    const void *a, *b;
    long long as, bs;                // stride of the axis that is not contiguous
    int I, J, K;
    int tiles_i, tiles_j;
    int splits, k_split;             // splits > 1: split s adds k in [s * k_split, (s + 1) * k_split) into partial[s][I][J]
    int avec, bvec;                  // 16-byte loads along the contiguous axis are aligned
    float* partial;
    void* c;
    long long cs;                    // c[i * cs + j]
    const void* bias;
    int bias_i;                      // the bias goes with i, not j (the product was turned over)
    int act;
    float slope;
    const void* res;
    long long ri, rj;
    void* pre;
    long long pi, pj;
    int c16;                         // rows of c, res and pre lie on 16 bytes, j contiguous
};

__device__ inline float act_of(float z, int act, float slope) {
    switch (act) {
        case AIPT_ACT_LEAKY: return z > 0.f ? z : z * slope;
        case AIPT_ACT_SILU: return z / (1.f + expf(-z));
        case AIPT_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678f));
    }
    return z;
}
__device__ inline float act_slope_of(float z, int act, float slope) {
    switch (act) {
        case AIPT_ACT_LEAKY: return z > 0.f ? 1.f : slope;
        case AIPT_ACT_SILU: {
            const float e = 1.f / (1.f + expf(-z));
            return e * (1.f + z * (1.f - e));
        }
        case AIPT_ACT_GELU: return 0.5f * (1.f + erff(z * 0.70710678f)) + z * expf(-0.5f * z * z) * 0.39894228f;
    }
    return 1.f;
}

template <typename T> __device__ inline void epilogue(const GemmArgs& g, int i, int j, float z) {
    if (g.bias) z += (float)((const T*)g.bias)[g.bias_i ? i : j];
    if (g.pre) ((T*)g.pre)[i * g.pi + j * g.pj] = (T)z;
    float y = act_of(z, g.act, g.slope);
    if (g.res) y += (float)((const T*)g.res)[i * g.ri + j * g.rj];
    ((T*)g.c)[i * g.cs + j] = (T)y;
}

// ---- any sizes, strides and alignment: 64 x 64 tiles, a step of 128 bytes of k, guarded loads through registers.
// LDS: rows of 128 bytes of k, its eight 16-byte chunks at chunk ^ (row & 7), so that the 16 rows a wave reads together lie on all banks.
template <typename T> struct Mac;
template <> struct Mac<bf16> {
    static __device__ inline f32x4 go(const Chunk<bf16>& a, const Chunk<bf16>& b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8*)&a, *(const bf16x8*)&b, c, 0, 0, 0);
    }
};
template <> struct Mac<f16> {
    static __device__ inline f32x4 go(const Chunk<f16>& a, const Chunk<f16>& b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(*(const f16x8*)&a, *(const f16x8*)&b, c, 0, 0, 0);
    }
};
template <> struct Mac<float> {      // k runs 0, 4, 8, 12 (one of each lane group's four), then 1, 5, ...: any order is a sum
    static __device__ inline f32x4 go(const Chunk<float>& a, const Chunk<float>& b, f32x4 c) {
#pragma unroll
        for (int q = 0; q < 4; q++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[q], b.v[q], c, 0, 0, 0);
        return c;
    }
};

constexpr int GT = 64;               // tile of the general kernel

// 16 bytes of the operand's tile into registers: K contiguous: row r, elements k .. ; else row r .. , one k
template <typename T, bool KC>
__device__ inline Chunk<T> fetch(const T* p, long long stride, int rows, int K, int r, int k, bool vec) {
    constexpr int E = 16 / sizeof(T);
    Chunk<T> q;
#pragma unroll
    for (int e = 0; e < E; e++) q.v[e] = (T)0.f;
    const int n = KC ? K - k : rows - r;                     // elements that exist
    if ((KC ? rows - r : K - k) <= 0 || n <= 0) return q;
    const T* s = KC ? p + r * stride + k : p + k * stride + r;
    if (vec && n >= E) return *(const Chunk<T>*)s;
#pragma unroll
    for (int e = 0; e < E; e++) if (e < n) q.v[e] = s[e];
    return q;
}

template <typename T, bool AK, bool BK>
__global__ __launch_bounds__(256) void gemm_any(const GemmArgs g) {
    constexpr int E = 16 / sizeof(T), KS = 8 * E;            // elements of a chunk, of a step
    __shared__ Chunk<T> lds[2][GT * 8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int job = blockIdx.x;
    const int split = job % g.splits; job /= g.splits;
    const int i0 = job / g.tiles_j * GT, j0 = job % g.tiles_j * GT;
    const int k0 = split * g.k_split, k1 = min(g.K, k0 + g.k_split);
    f32x4 acc[2][2] = {};
    const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
    for (int k = k0; k < k1; k += KS) {
#pragma unroll
        for (int side = 0; side < 2; side++) {
            const bool kc = side ? BK : AK;
            const T* p = (const T*)(side ? g.b : g.a);
            const long long st = side ? g.bs : g.as;
            const int base = side ? j0 : i0, rows = side ? g.J : g.I;
            const bool vec = side ? g.bvec : g.avec;
            T* t = (T*)lds[side];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const int id = tid + n * 256;                // 512 chunks of a tile
                if (kc) {
                    const int r = id >> 3, c = id & 7;
                    lds[side][r * 8 + (c ^ (r & 7))] = fetch<T, true>(p, st, rows, k1, base + r, k + c * E, vec);
                } else {
                    constexpr int RC = GT / E;               // chunks along the rows
                    const int kk = id / RC, r = id % RC * E;
                    const Chunk<T> q = fetch<T, false>(p, st, rows, k1, base + r, k + kk, vec);
#pragma unroll
                    for (int e = 0; e < E; e++) t[(r + e) * KS + ((kk / E) ^ ((r + e) & 7)) * E + kk % E] = q.v[e];
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Chunk<T> fa[2], fb[2];
            const int c = s * 4 + (lane >> 4);
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int ra = wi + x * 16 + (lane & 15), rb = wj + x * 16 + (lane & 15);
                fa[x] = lds[0][ra * 8 + (c ^ (ra & 7))];
                fb[x] = lds[1][rb * 8 + (c ^ (rb & 7))];
            }
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int y = 0; y < 2; y++) acc[x][y] = Mac<T>::go(fb[y], fa[x], acc[x][y]);     // lane: i = lane % 16, j = lane / 16 * 4 ..
        }
        __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
        for (int y = 0; y < 2; y++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = i0 + wi + x * 16 + (lane & 15), j = j0 + wj + y * 16 + (lane >> 4) * 4 + e;
                if (i < g.I && j < g.J) {
                    if (g.splits > 1) g.partial[((long long)split * g.I + i) * g.J + j] = acc[x][y][e];
                    else epilogue<T>(g, i, j, acc[x][y][e]);
                }
            }
}

// ---- 16-bit types, lines on 16 bytes: tiles of TI x TJ, fed without a pause.
// A step is 32 of k (64 bytes).  ST steps of both operands lie in LDS, loaded there directly (buffer loads to LDS, 16 bytes a lane), ST - 1
// steps ahead of their use; the fragments of a step are read into registers while the matrix instructions of the step before run.  One
// barrier a step: behind it every wave has its fragments of step t, so that t's LDS is free for t + ST, and step t + 1 is visible.
//   k contiguous:    rows of 64 bytes, 16-byte chunk c of row r at c ^ (r / 4 % 4): the 16 rows a read takes together lie on all banks
//   rows contiguous: 32 lines (k) of the tile's rows, 32-byte chunk c of line k at c ^ (k % 4 + k / 8 % 2 * 4), read by the transposing
//                    LDS load (16 lanes x 4 elements: lines 4q .. 4q + 3, 16 rows -> each lane its row's four)
// Lines beyond the operand are clamped to its last one (their results are not stored), steps beyond k read as zero (beyond num_records).
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
#define AIPT_LDS __attribute__((address_space(3)))

// The accumulators are pinned to accumulation registers in place: with the builtin the compiler keeps a part of 64 of them in vector
// registers and moves it to and fro each step (0.84 of 1.3 PFLOP/s).  settle() stands between these instructions and everything else that
// touches an accumulator: the compiler does not know that they are matrix instructions, whose results and sources want wait states.
template <typename T> struct Frag;
template <> struct Frag<bf16> {
    using V = bf16x8;
    static __device__ inline void mac(V a, V b, f32x4& c) { asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b)); }
};
template <> struct Frag<f16> {
    using V = f16x8;
    static __device__ inline void mac(V a, V b, f32x4& c) { asm("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b)); }
};
template <int N> __device__ inline void settle(f32x4* acc) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (i == 0) asm volatile("s_nop 15\n\ts_nop 15" : "+a"(acc[i]));
        else asm volatile("" : "+a"(acc[i]));
    }
}

// loads of one operand's part of a step: R rows x 32 k = R * 64 bytes, split over NT threads
template <bool KC, int R, int NT> struct TileLoad {
    static constexpr int L = R * 4 / NT;
    unsigned off[L];
    int kof[L];                      // the k of this lane's chunk within a step
    const char* base;
    long long step;                  // bytes to the next step
    __device__ inline void init(const void* p, long long stride, int r0, int rows, int k0, int tid) {
        // (a line's contiguous rows come in eights: rows is a multiple of 8, or its lines are padded to one)
        base = (const char*)p + (KC ? ((long long)r0 * stride + k0) * 2 : ((long long)k0 * stride + r0) * 2);
        step = KC ? 64 : 64 * stride;
        const int last = KC ? rows - 1 - r0 : ((rows + 7) & ~7) - 8 - r0;
#pragma unroll
        for (int i = 0; i < L; i++) {
            const int q = i * NT + tid;
            if (KC) {
                const int r = q >> 2, c = (q & 3) ^ ((r >> 2) & 3);
                off[i] = (unsigned)min(r, last) * (unsigned)(stride * 2) + c * 16;
                kof[i] = c * 8;
            } else {
                const int k = q / (R / 8), c = q % (R / 8);
                const int mn = (((c >> 1) ^ ((k & 3) | ((k >> 1) & 4))) * 2 + (c & 1)) * 8;
                off[i] = (unsigned)k * (unsigned)(stride * 2) + (unsigned)min(mn, last) * 2;
                kof[i] = k;
            }
        }
    }
    // where step t lies; load i of it, `left` of k being left
    __device__ inline __amdgpu_buffer_rsrc_t at(int t) const { return __builtin_amdgcn_make_buffer_rsrc((void*)(base + t * step), 0, 0x7fffffff, 0x00027000); }
    __device__ inline void one(int i, __amdgpu_buffer_rsrc_t rs, int left, AIPT_LDS char* lds, int wave) const {
        const unsigned o = kof[i] < left ? off[i] : 0x80000000u;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (AIPT_LDS void*)(lds + (i * NT + wave * 64) * 16), 16, o, 0, 0, 0);
    }
};

// fragments of N x 16 rows from r0 on, 32 k
template <typename T, bool KC, int R, int N> struct TileRead {
    int at[KC ? 1 : N][2];
    __device__ inline void init(int r0, int lane) {
        if constexpr (KC) {
            const int r = r0 + (lane & 15);
            at[0][0] = r * 64 + (((lane >> 4) ^ ((r >> 2) & 3)) * 16);
        } else {
#pragma unroll
            for (int n = 0; n < N; n++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int k = (lane >> 4) * 8 + h * 4 + ((lane & 15) >> 2);
                    at[n][h] = k * R * 2 + (((r0 / 16 + n) ^ ((k & 3) | ((k >> 1) & 4))) * 32) + (lane & 3) * 8;
                }
        }
    }
    __device__ inline typename Frag<T>::V one(int n, AIPT_LDS char* lds) const {
        using V = typename Frag<T>::V;
        if constexpr (KC) return *(AIPT_LDS V*)(lds + at[0][0] + n * 1024);
        else {
            union { i16x4 h[2]; V v; } u;
            u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((AIPT_LDS i16x4*)(lds + at[n][0]));
            u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((AIPT_LDS i16x4*)(lds + at[n][1]));
            return u.v;
        }
    }
};

// eight neighbours of a row: bias, activation, residual, 16-byte stores
template <typename T, int ACT> __device__ inline void epilogue8(const GemmArgs& g, int i, int j, float* z, const float* bias_j) {
    float b[8];
    if (g.bias_i) {
        const float v = g.bias ? (float)((const T*)g.bias)[i] : 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) b[e] = v;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) b[e] = bias_j[e];
    }
    Chunk<T> q;
#pragma unroll
    for (int e = 0; e < 8; e++) z[e] += b[e];
    if (g.pre) {
#pragma unroll
        for (int e = 0; e < 8; e++) q.v[e] = (T)z[e];
        *(Chunk<T>*)((T*)g.pre + i * g.pi + j) = q;
    }
#pragma unroll
    for (int e = 0; e < 8; e++) z[e] = act_of(z[e], ACT, g.slope);
    if (g.res) {
        const Chunk<T> r = *(const Chunk<T>*)((const T*)g.res + i * g.ri + j);
#pragma unroll
        for (int e = 0; e < 8; e++) z[e] += (float)r.v[e];
    }
#pragma unroll
    for (int e = 0; e < 8; e++) q.v[e] = (T)z[e];
    *(Chunk<T>*)((T*)g.c + i * g.cs + j) = q;
}

template <typename T, bool AK, bool BK, int TI, int TJ, int WI, int WJ, int ST>
__global__ __launch_bounds__(WI * WJ * 64, 1) void gemm_tile(const GemmArgs g) {
    constexpr int NT = WI * WJ * 64, WTI = TI / WI, WTJ = TJ / WJ, FI = WTI / 16, FJ = WTJ / 16, SB = (TI + TJ) * 64;
    constexpr int SLAB = WTI < 64 ? WTI : 64;                // rows of a wave's results that go through LDS at a time
    constexpr int BYTES = ST * SB > WI * WJ * SLAB * WTJ * 4 ? ST * SB : WI * WJ * SLAB * WTJ * 4;
    __shared__ __attribute__((aligned(1024))) char lds_[BYTES];
    AIPT_LDS char* lds = (AIPT_LDS char*)lds_;
    using V = typename Frag<T>::V;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // workgroups go round the eight XCDs: each XCD takes a run of neighbouring tiles, which share operands in its L2 ...
    const int total = gridDim.x, per = total >> 3, extra = total & 7, x = blockIdx.x & 7;
    int job = (x < extra ? x * (per + 1) : extra * (per + 1) + (x - extra) * per) + (blockIdx.x >> 3);
    const int tiles = g.tiles_i * g.tiles_j, split = job / tiles;
    job -= split * tiles;
    // ... in columns of 8 tiles
    const int band = 8 * g.tiles_j, b0 = job / band * 8, bh = min(8, g.tiles_i - b0);
    const int i0 = (b0 + (job % band) % bh) * TI, j0 = (job % band) / bh * TJ;
    const int k0 = split * g.k_split, k1 = min(g.K, k0 + g.k_split), n = (k1 - k0 + 31) >> 5;

    TileLoad<AK, TI, NT> la;
    TileLoad<BK, TJ, NT> lb;
    la.init(g.a, g.as, i0, g.I, k0, tid);
    lb.init(g.b, g.bs, j0, g.J, k0, tid);
    const int wi = wave / WJ * WTI, wj = wave % WJ * WTJ;
    TileRead<T, AK, TI, FI> ra;
    TileRead<T, BK, TJ, FJ> rb;
    ra.init(wi, lane);
    rb.init(wj, lane);
    constexpr int LA = decltype(la)::L, LB = decltype(lb)::L, L = LA + LB;
    f32x4 acc[FI][FJ] = {};
    settle<FI * FJ>(&acc[0][0]);
    V a0[FI], b0f[FJ], a1[FI], b1f[FJ];
#pragma unroll
    for (int t = 0; t < ST; t++) {
        const auto sa = la.at(t), sb = lb.at(t);
#pragma unroll
        for (int i = 0; i < L; i++)
            if (i < LA) la.one(i, sa, k1 - k0 - t * 32, lds + t * SB, wave);
            else lb.one(i - LA, sb, k1 - k0 - t * 32, lds + t * SB + TI * 64, wave);
    }
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((ST - 1) * L) : "memory");
#pragma unroll
    for (int p = 0; p < FI; p++) a0[p] = ra.one(p, lds);
#pragma unroll
    for (int q = 0; q < FJ; q++) b0f[q] = rb.one(q, lds + TI * 64);
    int slot = 0;
    // The order is the program's, not the scheduler's (which would read the next fragments behind the last product, into the registers
    // that these leave, and so wait for them): rows of FJ products, the reads of the next fragments between the first half of the rows, the
    // loads of a later step between the second half.
    auto step = [&](int t, V* a, V* b, V* an, V* bn) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((ST - 2) * L) : "memory");
        AIPT_LDS char* into = lds + slot * SB;
        slot = slot == ST - 1 ? 0 : slot + 1;
        AIPT_LDS char* from = lds + slot * SB;
        const auto sa = la.at(t + ST), sb = lb.at(t + ST);
        const int left = k1 - k0 - (t + ST) * 32;
        constexpr int H = FI / 2, R = (FI + FJ + H - 1) / H, G = (L + H - 1) / H;
#pragma unroll
        for (int p = 0; p < FI; p++) {
            if (p < H) {
#pragma unroll
                for (int r = p * R; r < (p + 1) * R && r < FI + FJ; r++) {
                    if (r < FI) an[r] = ra.one(r, from);
                    else bn[r - FI] = rb.one(r - FI, from + TI * 64);
                }
            } else {
#pragma unroll
                for (int i = (p - H) * G; i < (p - H + 1) * G && i < L; i++)
                    if (i < LA) la.one(i, sa, left, into, wave);
                    else lb.one(i - LA, sb, left, into + TI * 64, wave);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int q = 0; q < FJ; q++) Frag<T>::mac(b[q], a[p], acc[p][q]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    for (int t = 0; t < n; t += 2) {                         // (an odd last step adds zeros)
        step(t, a0, b0f, a1, b1f);
        step(t + 1, a1, b1f, a0, b0f);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    settle<FI * FJ>(&acc[0][0]);

    // results: through a slab of LDS of the wave's own (chunk c of row r at c ^ (r % 16)), so that rows are stored in 16-byte pieces
    AIPT_LDS char* slab = lds + wave * (SLAB * WTJ * 4);
    constexpr int LR = WTJ / 8, RPI = 64 / LR;               // lanes of a row, rows of an instruction
    const int j = j0 + wj + lane % LR * 8;
    const bool whole = j + 8 <= g.J && g.c16;
    float bias_j[8];
#pragma unroll
    for (int e = 0; e < 8; e++) bias_j[e] = g.bias && !g.bias_i && g.splits == 1 && j + e < g.J ? (float)((const T*)g.bias)[j + e] : 0.f;
#pragma unroll
    for (int s = 0; s < WTI / SLAB; s++) {
#pragma unroll
        for (int p = 0; p < SLAB / 16; p++)
#pragma unroll
            for (int q = 0; q < FJ; q++) {
                const int r = p * 16 + (lane & 15), c = q * 4 + (lane >> 4);
                *(AIPT_LDS f32x4*)(slab + r * (WTJ * 4) + ((c ^ (r & 15)) * 16)) = acc[s * (SLAB / 16) + p][q];
            }
        auto rows = [&](auto done) {
            for (int r = lane / LR; r < SLAB; r += RPI) {
                const int i = i0 + wi + s * SLAB + r;
                if (i >= g.I || j >= g.J) continue;
                float z[8];
                const int c = lane % LR * 2;
                *(f32x4*)z = *(AIPT_LDS f32x4*)(slab + r * (WTJ * 4) + ((c ^ (r & 15)) * 16));
                *(f32x4*)(z + 4) = *(AIPT_LDS f32x4*)(slab + r * (WTJ * 4) + (((c + 1) ^ (r & 15)) * 16));
                done(i, z);
            }
        };
        if (g.splits > 1) rows([&](int i, float* z) {
            float* o = g.partial + ((long long)split * g.I + i) * g.J + j;
#pragma unroll
            for (int e = 0; e < 8; e++) if (j + e < g.J) o[e] = z[e];
        });
        else if (!whole) rows([&](int i, float* z) {
#pragma unroll
            for (int e = 0; e < 8; e++) if (j + e < g.J) epilogue<T>(g, i, j + e, z[e]);
        });
        else if (g.act == AIPT_ACT_NONE) rows([&](int i, float* z) { epilogue8<T, AIPT_ACT_NONE>(g, i, j, z, bias_j); });
        else if (g.act == AIPT_ACT_LEAKY) rows([&](int i, float* z) { epilogue8<T, AIPT_ACT_LEAKY>(g, i, j, z, bias_j); });
        else if (g.act == AIPT_ACT_SILU) rows([&](int i, float* z) { epilogue8<T, AIPT_ACT_SILU>(g, i, j, z, bias_j); });
        else rows([&](int i, float* z) { epilogue8<T, AIPT_ACT_GELU>(g, i, j, z, bias_j); });
    }
}

// the splits of a long contraction, added in order, and the epilogue
template <typename T>
__global__ __launch_bounds__(256) void gemm_join(const GemmArgs g) {
    const long long n = (long long)g.I * g.J;
    for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < n; at += (long long)gridDim.x * 256) {
        float s = 0;
        for (int k = 0; k < g.splits; k++) s += g.partial[k * n + at];
        epilogue<T>(g, (int)(at / g.J), (int)(at % g.J), s);
    }
}

// ---- dz = dy * act'(z), rounded to the element type, and its sums over rows: both read dy once.  Tiles of 64 (contiguous axis) x 64.
struct DzArgs {
    const void *dy, *z;
    void* dz;
    float* part;                     // [row tiles][N] sums over 64 rows, or NULL
    long long dyi, dyj, zi, zj, dzi, dzj;
    int M, N, tiles_n, turned;       // turned: rows are the contiguous axis
    int line;                        // dz's lines, with their padding (of zeros)
    int act;
    float slope;
};
template <typename T>
__global__ __launch_bounds__(256) void act_backward(const DzArgs g) {
    __shared__ float lds[64][65];
    const int m0 = (int)(blockIdx.x / g.tiles_n) * 64, n0 = (int)(blockIdx.x % g.tiles_n) * 64;
    const int x = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int y = w; y < 64; y += 4) {
        const int m = m0 + (g.turned ? x : y), n = n0 + (g.turned ? y : x);
        float d = 0;
        if (m < g.M && n < g.N) {
            d = (float)((const T*)g.dy)[m * g.dyi + n * g.dyj];
            if (g.act != AIPT_ACT_NONE) d *= act_slope_of((float)((const T*)g.z)[m * g.zi + n * g.zj], g.act, g.slope);
        }
        if (g.dz && (g.turned ? n < g.N && m < g.line : m < g.M && n < g.line)) ((T*)g.dz)[m * g.dzi + n * g.dzj] = (T)d;
        lds[g.turned ? x : y][g.turned ? y : x] = d;
    }
    if (!g.part) return;
    __syncthreads();
    float s = 0;
    for (int y = w; y < 64; y += 4) s += lds[y][x];
    __syncthreads();
    lds[w][x] = s;
    __syncthreads();
    if (w == 0 && n0 + x < g.N) g.part[(long long)(m0 / 64) * g.N + n0 + x] = (lds[0][x] + lds[1][x]) + (lds[2][x] + lds[3][x]);
}
struct SumArgs {
    const float* part;
    void* out;
    int parts, N;
};
template <typename T>
__global__ __launch_bounds__(256) void sum_parts(const SumArgs g) {
    __shared__ float lds[4][64];
    const int x = threadIdx.x & 63, w = threadIdx.x >> 6, n = blockIdx.x * 64 + x;
    float s = 0;
    if (n < g.N) for (int p = w; p < g.parts; p += 4) s += g.part[(long long)p * g.N + n];
    lds[w][x] = s;
    __syncthreads();
    if (w == 0 && n < g.N) ((T*)g.out)[n] = (T)((lds[0][x] + lds[1][x]) + (lds[2][x] + lds[3][x]));
}

struct FillArgs { unsigned short* p; size_t n; };
__global__ __launch_bounds__(256) void fill_zero(const FillArgs g) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < g.n; i += (size_t)gridDim.x * 256) g.p[i] = 0;
}
hipError_t zero_fill(hipStream_t st, const void* data, size_t bytes) {
    if (!data || !bytes) return hipSuccess;
    return launch(fill_zero, std::min<size_t>((bytes / 2 + 255) / 256, 4096), 256, 0, st, FillArgs{(unsigned short*)data, bytes / 2});
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------

static_assert(sizeof(aipt_linear_args) == 168 && sizeof(aipt_linear_grad_args) == 192, "argument records (api.py packs them by field)");

constexpr long long SIZE_MAX_DIM = 0x7fffffffll - 4096;

// an operand or result as the kernels take it: which axis is contiguous, and the other one's stride
struct View {
    char* p;
    long long ri, rj;                // strides of the first and the second axis
    bool second;                     // the second axis is the contiguous one
    long long other;                 // the stride of the other
    bool padded = false;             // lines are padded with zeros to a multiple of 16 bytes
};
static View view_of(const aipt_matrix& m, long long n0, long long n1) {
    View v{(char*)m.data, m.row_stride, m.col_stride, false, 0};
    // a stride of an axis of one element is never used: take what makes the other the contiguous one
    const bool j1 = v.rj == 1 || n1 <= 1, i1 = v.ri == 1 || n0 <= 1;
    v.second = j1 && !(i1 && n1 <= 1 && n0 > 1 && v.ri == 1);
    v.other = v.second ? (n0 <= 1 ? n1 : v.ri) : (n1 <= 1 ? n0 : v.rj);
    return v;
}
static bool strides_ok(const aipt_matrix& m, long long n0, long long n1, bool out) {
    const bool j1 = m.col_stride == 1 || n1 <= 1, i1 = m.row_stride == 1 || n0 <= 1;
    if (!j1 && !i1) return false;
    const long long hi = 1ll << 40;
    for (int a = 0; a < 2; a++) {
        const long long s = a ? m.col_stride : m.row_stride, n = a ? n1 : n0;
        if (n > 1 && (s < 0 || s > hi)) return false;
    }
    if (out) {
        if (n0 > 1 && n1 > 1) return (m.col_stride == 1 && m.row_stride >= n1) || (m.row_stride == 1 && m.col_stride >= n0);
        if (n0 > 1) return m.row_stride >= 1;
        if (n1 > 1) return m.col_stride >= 1;
    }
    return true;
}
static Extent extent_of(const aipt_matrix& m, long long n0, long long n1, int es) {
    if (!m.data || n0 <= 0 || n1 <= 0) return {};
    const View v = view_of(m, n0, n1);
    if (v.second) return {v.p, n0, ((n1 > 1 ? (n1 - 1) * v.rj : 0) + 1) * es, (n0 > 1 ? v.ri : 0) * es};
    return {v.p, n1, ((n0 > 1 ? (n0 - 1) * v.ri : 0) + 1) * es, (n1 > 1 ? v.rj : 0) * es};
}

struct Plan {                        // a product as it will be launched, and the workspace it wants
    GemmArgs g = {};
    bool ak = true, bk = true;
    int tile = 0;                    // 0: gemm_any; else gemm_tile of this size
    unsigned threads = 256;
    size_t partial_bytes = 0, blocks = 0;
    bool fits = true;
};

// C[i][j] = sum_k A[i][k] B[j][k]; A (I x K) and B (J x K) by their strides; the result's j axis contiguous
static Plan plan_gemm(int type, const View& a, const View& b, long long I, long long J, long long K) {
    Plan p;
    const int es = type_bytes(type), E = 16 / es, ks = 8 * E;
    p.g.a = a.p; p.g.b = b.p;
    p.ak = a.second; p.bk = b.second;
    p.g.as = a.other; p.g.bs = b.other;
    p.g.I = (int)I; p.g.J = (int)J; p.g.K = (int)K;
    p.g.avec = !((uintptr_t)a.p & 15) && (a.other % E == 0);
    p.g.bvec = !((uintptr_t)b.p & 15) && (b.other % E == 0);
    // gemm_tile wants 16-bit elements, lines on 16 bytes that hold whole 16-byte chunks, and a tile's lines within 31 bits of its first
    auto lines_ok = [&](const View& v, bool vec, long long len) { return vec && (v.padded || len % E == 0) && v.other * 2 * 256 < (1ll << 31); };
    if (es == 2 && K >= 32 && lines_ok(a, p.g.avec, a.second ? K : I) && lines_ok(b, p.g.bvec, b.second ? K : J)) p.tile = 256;
    const int ts = p.tile ? p.tile : GT;
    p.g.tiles_i = (int)((I + ts - 1) / ts); p.g.tiles_j = (int)((J + ts - 1) / ts);
    const long long tiles = (long long)p.g.tiles_i * p.g.tiles_j, steps = (K + ks - 1) / ks;
    // few tiles and a long contraction: split it until some 512 workgroups (two a CU) run, none with fewer than 4 steps
    long long splits = 1;
    const long long want = p.tile ? 256 : 512;
    if (tiles > 0 && tiles < want) splits = std::max(1ll, std::min(want / tiles, steps / 4));
    const long long per = splits > 1 ? (steps + splits - 1) / splits : std::max(1ll, steps);
    splits = std::max(1ll, (steps + per - 1) / per);
    p.g.splits = (int)splits;
    p.g.k_split = (int)std::min<long long>(per * ks, 0x7fffffffll - ks);
    p.blocks = (size_t)(tiles * splits);
    p.fits = grid_fits(p.blocks, 256);
    if (splits > 1) p.partial_bytes = (size_t)splits * I * J * sizeof(float);
    return p;
}

template <typename T> static void (*gemm_of(const Plan& p))(GemmArgs) {
    if constexpr (sizeof(T) == 2) {
        if (p.tile) return p.ak ? (p.bk ? gemm_tile<T, true, true, 256, 256, 2, 2, 4> : gemm_tile<T, true, false, 256, 256, 2, 2, 4>)
                                : (p.bk ? gemm_tile<T, false, true, 256, 256, 2, 2, 4> : gemm_tile<T, false, false, 256, 256, 2, 2, 4>);
    }
    return p.ak ? (p.bk ? gemm_any<T, true, true> : gemm_any<T, true, false>) : (p.bk ? gemm_any<T, false, true> : gemm_any<T, false, false>);
}
// whether the epilogue may move 16 bytes at a time
static int rows16(int es, const GemmArgs& g) {
    const long long e = 16 / es;
    return !(((uintptr_t)g.c | (uintptr_t)g.res | (uintptr_t)g.pre) & 15) && g.cs % e == 0 && (!g.res || (g.rj == 1 && g.ri % e == 0)) && (!g.pre || (g.pj == 1 && g.pi % e == 0));
}

template <typename T> static hipError_t run_gemm_t(hipStream_t st, Plan& p, void* ws) {
    if (!p.blocks) return hipSuccess;
    p.g.partial = (float*)ws;
    p.g.c16 = rows16(sizeof(T), p.g);
    hipError_t e = launch(gemm_of<T>(p), p.blocks, 256, 0, st, p.g);
    if (e == hipSuccess && p.g.splits > 1)
        e = launch(gemm_join<T>, std::min<size_t>(((size_t)p.g.I * p.g.J + 255) / 256, 4096), 256, 0, st, p.g);
    return e;
}
static hipError_t run_gemm(int type, hipStream_t st, Plan& p, void* ws) {
    return type == AIPT_TYPE_F32 ? run_gemm_t<float>(st, p, ws) : type == AIPT_TYPE_BF16 ? run_gemm_t<bf16>(st, p, ws) : run_gemm_t<f16>(st, p, ws);
}

// the forward product: turned over (C^T = w x^T) where y's rows are the contiguous axis
static Plan plan_forward(const aipt_linear_args* a) {
    const View x = view_of(a->x, a->m, a->k), w = view_of(a->w, a->n, a->k), y = view_of(a->y, a->m, a->n);
    const bool turn = !y.second;
    Plan p = turn ? plan_gemm(a->type, w, x, a->n, a->m, a->k) : plan_gemm(a->type, x, w, a->m, a->n, a->k);
    GemmArgs& g = p.g;
    g.c = a->y.data; g.cs = y.other;
    g.bias = a->bias; g.bias_i = turn; g.act = a->act; g.slope = a->slope;
    g.res = a->residual.data; g.ri = a->residual.row_stride; g.rj = a->residual.col_stride;
    g.pre = a->preact.data; g.pi = a->preact.row_stride; g.pj = a->preact.col_stride;
    if (turn) { std::swap(g.ri, g.rj); std::swap(g.pi, g.pj); }
    return p;
}

struct GradPlan {
    Plan dx, dw;
    DzArgs dz = {};
    bool want_dx = false, want_dw = false, want_db = false, make_dz = false;
    size_t dz_bytes = 0, part_bytes = 0, gemm_bytes = 0, dz_blocks = 0;
    size_t bytes() const { return dz_bytes + part_bytes + gemm_bytes; }
};
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
static GradPlan plan_backward(const aipt_linear_grad_args* a, char* ws) {
    GradPlan p;
    const int es = type_bytes(a->type), E = 16 / es;
    p.want_dx = a->dx.data && a->m > 0 && a->k > 0;
    p.want_dw = a->dw.data && a->n > 0 && a->k > 0;
    p.want_db = a->dbias && a->n > 0;
    const View dy = view_of(a->dy, a->m, a->n), z = view_of(a->preact, a->m, a->n);
    p.make_dz = a->act != AIPT_ACT_NONE && (p.want_dx || p.want_dw);
    View d = dy;
    if (p.make_dz) {                 // laid out like dy, with lines a multiple of 16 bytes apart
        const long long line = dy.second ? a->n : a->m, lines = dy.second ? a->m : a->n, ld = (line + E - 1) / E * E;
        p.dz_bytes = up256((size_t)(lines * ld) * es);
        p.dz.line = (int)ld;
        d = {ws, dy.second ? ld : 1, dy.second ? 1 : ld, dy.second, ld, true};
    }
    const long long tm = (a->m + 63) / 64, tn = (a->n + 63) / 64;
    if (p.want_db) p.part_bytes = up256((size_t)tm * a->n * sizeof(float));
    if (p.make_dz || p.want_db) {
        DzArgs& g = p.dz;
        g.dy = a->dy.data; g.z = a->preact.data; g.dz = p.make_dz ? d.p : nullptr;
        g.part = p.want_db ? (float*)(ws + p.dz_bytes) : nullptr;
        g.dyi = dy.ri; g.dyj = dy.rj; g.zi = z.ri; g.zj = z.rj; g.dzi = d.ri; g.dzj = d.rj;
        g.M = (int)a->m; g.N = (int)a->n; g.tiles_n = (int)tn; g.turned = !dy.second;
        g.act = a->act; g.slope = a->slope;
        p.dz_blocks = (size_t)(tm * tn);
    }
    auto flip = [](View v) { std::swap(v.ri, v.rj); v.second = !v.second; return v; };
    if (p.want_dx) {                 // dx[m][k] = sum_n dz[m][n] w[n][k]
        const View w = view_of(a->w, a->n, a->k), o = view_of(a->dx, a->m, a->k);
        p.dx = o.second ? plan_gemm(a->type, d, flip(w), a->m, a->k, a->n) : plan_gemm(a->type, flip(w), d, a->k, a->m, a->n);
        p.dx.g.c = a->dx.data; p.dx.g.cs = o.other;
    }
    if (p.want_dw) {                 // dw[n][k] = sum_m dz[m][n] x[m][k]
        const View x = view_of(a->x, a->m, a->k), o = view_of(a->dw, a->n, a->k);
        p.dw = o.second ? plan_gemm(a->type, flip(d), flip(x), a->n, a->k, a->m) : plan_gemm(a->type, flip(x), flip(d), a->k, a->n, a->m);
        p.dw.g.c = a->dw.data; p.dw.g.cs = o.other;
    }
    p.gemm_bytes = up256(std::max(p.want_dx ? p.dx.partial_bytes : 0, p.want_dw ? p.dw.partial_bytes : 0));
    return p;
}

static int linear_check(aipt_ctx* ctx, const char* me, int type, int act, float slope, int reserved, long long m, long long n, long long k) {
    if (reserved) return fail(ctx, AIPT_E_INVALID, "%s: reserved is not 0", me);
    if (!type_ok(type)) return fail(ctx, AIPT_E_INVALID, "%s: type %d", me, type);
    if (act < AIPT_ACT_NONE || act > AIPT_ACT_GELU) return fail(ctx, AIPT_E_INVALID, "%s: act %d", me, act);
    if (slope != slope) return fail(ctx, AIPT_E_INVALID, "%s: slope is NaN", me);
    for (long long s : {m, n, k}) if (s < 0 || s > SIZE_MAX_DIM) return fail(ctx, AIPT_E_INVALID, "%s: sizes %lld x %lld x %lld", me, m, n, k);
    return AIPT_OK;
}
static int matrix_check(aipt_ctx* ctx, const char* me, const char* name, const aipt_matrix& q, long long n0, long long n1, int es, bool out, bool optional, bool pointers) {
    if (optional && !q.data) return AIPT_OK;
    if (pointers && !q.data && n0 > 0 && n1 > 0) return fail(ctx, AIPT_E_INVALID, "%s: %s is NULL", me, name);
    if (!strides_ok(q, n0, n1, out)) return fail(ctx, AIPT_E_INVALID, "%s: %s: strides (%lld, %lld) of %lld x %lld", me, name, q.row_stride, q.col_stride, n0, n1);
    if (!pointers) return AIPT_OK;
    if ((uintptr_t)q.data & (es - 1)) return fail(ctx, AIPT_E_INVALID, "%s: %s is misaligned", me, name);
    return AIPT_OK;
}

static int forward_check(aipt_ctx* ctx, const char* me, const aipt_linear_args* a, bool pointers) {
    if (!a) return fail(ctx, AIPT_E_INVALID, "%s: args is NULL", me);
    int rc = linear_check(ctx, me, a->type, a->act, a->slope, a->reserved, a->m, a->n, a->k);
    const int es = rc ? 0 : type_bytes(a->type);
    if (!rc) rc = matrix_check(ctx, me, "x", a->x, a->m, a->k, es, false, false, pointers);
    if (!rc) rc = matrix_check(ctx, me, "w", a->w, a->n, a->k, es, false, false, pointers);
    if (!rc) rc = matrix_check(ctx, me, "y", a->y, a->m, a->n, es, true, false, pointers);
    if (!rc) rc = matrix_check(ctx, me, "residual", a->residual, a->m, a->n, es, false, true, pointers);
    if (!rc) rc = matrix_check(ctx, me, "preact", a->preact, a->m, a->n, es, true, true, pointers);
    if (!rc && pointers && ((uintptr_t)a->bias & (es - 1))) rc = fail(ctx, AIPT_E_INVALID, "%s: bias is misaligned", me);
    return rc;
}
static int backward_check(aipt_ctx* ctx, const char* me, const aipt_linear_grad_args* a, bool pointers) {
    if (!a) return fail(ctx, AIPT_E_INVALID, "%s: args is NULL", me);
    int rc = linear_check(ctx, me, a->type, a->act, a->slope, a->reserved, a->m, a->n, a->k);
    const int es = rc ? 0 : type_bytes(a->type);
    if (!rc) rc = matrix_check(ctx, me, "dy", a->dy, a->m, a->n, es, false, false, pointers);
    if (!rc) rc = matrix_check(ctx, me, "x", a->x, a->m, a->k, es, false, !a->dw.data, pointers);
    if (!rc) rc = matrix_check(ctx, me, "w", a->w, a->n, a->k, es, false, !a->dx.data, pointers);
    if (!rc) rc = matrix_check(ctx, me, "preact", a->preact, a->m, a->n, es, false, a->act == AIPT_ACT_NONE, pointers);
    if (!rc) rc = matrix_check(ctx, me, "dx", a->dx, a->m, a->k, es, true, true, pointers);
    if (!rc) rc = matrix_check(ctx, me, "dw", a->dw, a->n, a->k, es, true, true, pointers);
    if (!rc && pointers && ((uintptr_t)a->dbias & (es - 1))) rc = fail(ctx, AIPT_E_INVALID, "%s: dbias is misaligned", me);
    return rc;
}

}  // namespace aipt

using aipt::fail;

extern "C" {

int aipt_linear_workspace(aipt_ctx* ctx, const aipt_linear_args* a, size_t* bytes) {
    if (!bytes) return fail(ctx, AIPT_E_INVALID, "aipt_linear_workspace: bytes is NULL");
    const int rc = aipt::forward_check(ctx, "aipt_linear_workspace", a, false);
    if (rc) return rc;
    *bytes = aipt::plan_forward(a).partial_bytes;
    return AIPT_OK;
}

int aipt_linear(aipt_ctx* ctx, const aipt_linear_args* a, void* d_workspace, size_t workspace_bytes) {
    const char* me = "aipt_linear";
    const int rc = aipt::forward_check(ctx, me, a, true);
    if (rc) return rc;
    const int es = aipt::type_bytes(a->type);
    aipt::Plan p = aipt::plan_forward(a);
    if (!p.fits) return fail(ctx, AIPT_E_INVALID, "%s: %lld x %lld has too many tiles", me, a->m, a->n);
    if (p.partial_bytes && (!d_workspace || workspace_bytes < p.partial_bytes || ((uintptr_t)d_workspace & 255)))
        return fail(ctx, AIPT_E_INVALID, "%s: workspace of %zu bytes, %zu are wanted, 256-byte aligned", me, workspace_bytes, p.partial_bytes);
    const aipt::Extent x = aipt::extent_of(a->x, a->m, a->k, es), w = aipt::extent_of(a->w, a->n, a->k, es), y = aipt::extent_of(a->y, a->m, a->n, es),
                       r = aipt::extent_of(a->residual, a->m, a->n, es), z = aipt::extent_of(a->preact, a->m, a->n, es), b = {(const char*)a->bias, 1, a->n * es, 0},
                       s = {(const char*)d_workspace, 1, (long long)p.partial_bytes, 0};
    const bool in_place = a->residual.data == a->y.data && a->residual.row_stride == a->y.row_stride && a->residual.col_stride == a->y.col_stride;
    for (const aipt::Extent& o : {y, z, s})
        for (const aipt::Extent& i : {x, w, b}) if (aipt::overlap(o, i)) return fail(ctx, AIPT_E_INVALID, "%s: an output overlaps an input", me);
    if ((!in_place && aipt::overlap(y, r)) || aipt::overlap(z, r) || aipt::overlap(s, r)) return fail(ctx, AIPT_E_INVALID, "%s: an output overlaps the residual", me);
    if (aipt::overlap(y, z) || aipt::overlap(y, s) || aipt::overlap(z, s)) return fail(ctx, AIPT_E_INVALID, "%s: outputs overlap", me);
    AIPT_NEED_CTX(ctx);
    if (!a->m || !a->n) return AIPT_OK;
    aipt::DeviceScope dev(ctx->device);
    AIPT_HIP(ctx, dev.err);
    AIPT_HIP(ctx, aipt::run_gemm(a->type, ctx->stream, p, d_workspace));
    return AIPT_OK;
}

int aipt_linear_backward_workspace(aipt_ctx* ctx, const aipt_linear_grad_args* a, size_t* bytes) {
    if (!bytes) return fail(ctx, AIPT_E_INVALID, "aipt_linear_backward_workspace: bytes is NULL");
    const int rc = aipt::backward_check(ctx, "aipt_linear_backward_workspace", a, false);
    if (rc) return rc;
    *bytes = aipt::plan_backward(a, nullptr).bytes();
    return AIPT_OK;
}

int aipt_linear_backward(aipt_ctx* ctx, const aipt_linear_grad_args* a, void* d_workspace, size_t workspace_bytes) {
    const char* me = "aipt_linear_backward";
    const int rc = aipt::backward_check(ctx, me, a, true);
    if (rc) return rc;
    const int es = aipt::type_bytes(a->type);
    aipt::GradPlan p = aipt::plan_backward(a, (char*)d_workspace);
    if ((p.want_dx && !p.dx.fits) || (p.want_dw && !p.dw.fits) || !aipt::grid_fits(p.dz_blocks, 256))
        return fail(ctx, AIPT_E_INVALID, "%s: %lld x %lld x %lld has too many tiles", me, a->m, a->n, a->k);
    if (p.bytes() && (!d_workspace || workspace_bytes < p.bytes() || ((uintptr_t)d_workspace & 255)))
        return fail(ctx, AIPT_E_INVALID, "%s: workspace of %zu bytes, %zu are wanted, 256-byte aligned", me, workspace_bytes, p.bytes());
    const aipt::Extent dy = aipt::extent_of(a->dy, a->m, a->n, es), none, x = a->dw.data ? aipt::extent_of(a->x, a->m, a->k, es) : none,
                       w = a->dx.data ? aipt::extent_of(a->w, a->n, a->k, es) : none, z = a->act ? aipt::extent_of(a->preact, a->m, a->n, es) : none,
                       dx = aipt::extent_of(a->dx, a->m, a->k, es), dw = aipt::extent_of(a->dw, a->n, a->k, es), db = {(const char*)a->dbias, 1, a->n * es, 0},
                       s = {(const char*)d_workspace, 1, (long long)p.bytes(), 0};
    const aipt::Extent out[] = {dx, dw, db, s};
    for (int o = 0; o < 4; o++) {
        for (const aipt::Extent& i : {dy, x, w, z}) if (aipt::overlap(out[o], i)) return fail(ctx, AIPT_E_INVALID, "%s: an output overlaps an input", me);
        for (int i = 0; i < o; i++) if (aipt::overlap(out[o], out[i])) return fail(ctx, AIPT_E_INVALID, "%s: outputs overlap", me);
    }
    AIPT_NEED_CTX(ctx);
    aipt::DeviceScope dev(ctx->device);
    AIPT_HIP(ctx, dev.err);
    const hipStream_t st = ctx->stream;
    const int t = a->type;
    if (p.dz_blocks)
        AIPT_HIP(ctx, aipt::launch(t == AIPT_TYPE_F32 ? aipt::act_backward<float> : t == AIPT_TYPE_BF16 ? aipt::act_backward<aipt::bf16> : aipt::act_backward<aipt::f16>, p.dz_blocks, 256, 0, st, p.dz));
    if (p.want_db) {
        if (a->m) AIPT_HIP(ctx, aipt::launch(t == AIPT_TYPE_F32 ? aipt::sum_parts<float> : t == AIPT_TYPE_BF16 ? aipt::sum_parts<aipt::bf16> : aipt::sum_parts<aipt::f16>, (size_t)((a->n + 63) / 64), 256, 0, st,
                                             aipt::SumArgs{p.dz.part, a->dbias, (int)((a->m + 63) / 64), (int)a->n}));
        else AIPT_HIP(ctx, aipt::zero_fill(st, a->dbias, (size_t)a->n * es));
    }
    char* gemm_ws = (char*)d_workspace + p.dz_bytes + p.part_bytes;
    if (p.want_dx) AIPT_HIP(ctx, aipt::run_gemm(t, st, p.dx, gemm_ws));
    if (p.want_dw) AIPT_HIP(ctx, aipt::run_gemm(t, st, p.dw, gemm_ws));
    return AIPT_OK;
}

}  // extern "C"
