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
    int turned;                      // gemm_rows: A and B are the result's j and i
    int cv;                          // elements that move together: 8 (rows of c, res and pre on 16 bytes, j contiguous), 9: 8 from anywhere on, or 1
};

// 1 / (1 + e^-z) by the chip's exponential and reciprocal (an ulp each): z is within 2^-24 |z| of what it should be in the exponent
__device__ inline float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f)); }
// The normal distribution below z, and e = e^(-z^2 / 2), which the slope wants too.  With a = |z| and t = 1 / (1 + p a), the tail e erfcx(a / sqrt 2) / 2 is
// e t P(t): P is a polynomial fitted (weighted least squares, the weights iterated until the largest error is least) for 0 <= a <= 16 by its RELATIVE
// error, so that what is small is right in its digits too, down to the end of fp32's range.  16-bit results: seven coefficients, 1.2e-6, and an
// exponent rounded in fp32 (a^2 2^-24): a fiftieth of fp16's half step at most, in some 20 instructions, which a tile's 256 results a lane feel.  Floats:
// ten, 8.3e-9, and the exponent with what its rounding lost: within 9 x 2^-24 of the result altogether (0.5 (1 + erff), the usual form, is off by 1e-5 of
// it at -3 and has no digits left at -5.5).
template <bool FLOAT> __device__ inline float below(float z, float& e) {
    constexpr float C = -0.72134752f, C_LO = -(float)(0.72134752044448170368 - 0.72134752f);      // -log2(e) / 2
    const float a = fminf(fabsf(z), 16.f), s = a * a, w = s * C;
    float q;
    e = __builtin_amdgcn_exp2f(w);
    if constexpr (FLOAT) {
        const float lost = fmaf(fmaf(a, a, -s), C, fmaf(s, C_LO, fmaf(s, C, -w)));
        e = fmaf(e, lost * 0.69314718f, e);
        const float t = __builtin_amdgcn_rcpf(fmaf(a, 0.38890873f, 1.f));
        constexpr float P[] = {
            0.155146554f, 0.15531975f, 0.129527479f, 0.100390859f, -0.0454047062f,
            0.177593619f, -0.420847416f, 0.385778248f, -0.166079387f, 0.0285749864f};
        q = P[9];
#pragma unroll
        for (int i = 8; i >= 0; i--) q = fmaf(q, t, P[i]);
        q = q * t * e;
    } else {
        const float t = __builtin_amdgcn_rcpf(fmaf(a, 0.36769553f, 1.f));
        constexpr float P[] = {
            0.146736786f, 0.145598784f, 0.136796817f, 0.0406556167f, 0.155492425f, -0.173597828f, 0.0483179614f};
        q = P[6];
#pragma unroll
        for (int i = 5; i >= 0; i--) q = fmaf(q, t, P[i]);
        q = q * t * e;
    }
    return z > 0.f ? 1.f - q : q;
}
template <typename T> __device__ inline float act_of(float z, int act, float slope) {
    float e;
    switch (act) {
        case AIPT_ACT_LEAKY: return z > 0.f ? z : z * slope;
        case AIPT_ACT_SILU: return z * sigmoid(z);
        case AIPT_ACT_GELU: return z * below<sizeof(T) == 4>(z, e);
    }
    return z;
}
template <typename T> __device__ inline float act_slope_of(float z, int act, float slope) {
    switch (act) {
        case AIPT_ACT_LEAKY: return z > 0.f ? 1.f : slope;
        case AIPT_ACT_SILU: {
            const float e = sigmoid(z);
            return e * (1.f + z * (1.f - e));
        }
        case AIPT_ACT_GELU: {
            float e;
            const float p = below<sizeof(T) == 4>(z, e);
            return fmaf(z, e * 0.39894228f, p);
        }
    }
    return 1.f;
}

template <typename T> __device__ inline void epilogue(const GemmArgs& g, int i, int j, float z) {
    if (g.bias) z += (float)((const T*)g.bias)[g.bias_i ? i : j];
    if (g.pre) ((T*)g.pre)[i * g.pi + j * g.pj] = (T)z;
    float y = act_of<T>(z, g.act, g.slope);
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
    const int k0 = split * g.k_split, k1 = (int)min((long long)g.K, (long long)k0 + g.k_split);
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

// ---- Lines on 16 bytes: tiles of TI x TJ, fed without a pause.
// A pair of steps is 128 bytes of k (64, or 32 floats): whole 128-byte lines of an operand with k contiguous (half lines cost the L2 as much as whole ones: 32 of k
// at a time ran at 1.15 PFLOP/s).  LDS is a ring of S slots, each one operand's part of a pair, loaded there directly (buffer loads to LDS, 16
// bytes a lane) in the order A(0) B(0) A(1) B(1) ...; the fragments of a step are read into registers while the matrix instructions of
// the step before run.  One barrier a pair, before its second step: behind it every wave has read all of pair P, whose slots are
// free for the loads S ahead of them, and pair P + 1 is visible.  4096^3 bf16 112 us (1.23 PFLOP/s) with both operands' k contiguous, 118 - 122
// otherwise (the library's product 95, 114 - 131); 8192 x 4096 by 16384 with gelu and two results 910.  The matrix pipes are busy 57 % of the cycles of that one
// (the library's product alone 89 %; under such a load the chip's power limit takes the clock down, to 1.7 - 2.0 GHz here and 1.4 - 1.8 there): what is left between
// the matrix instructions and the epilogue bound it.
//   k contiguous:    rows of 128 bytes, 16-byte chunk c of row r at c ^ (r / 2 % 8): the 16 rows a read takes together lie on all banks
//   rows contiguous: 64 lines (k) of the tile's rows, 32-byte group c of line k at c ^ (k % 4 + k / 8 % 2 * 4), read by the transposing
//                    LDS load (16 lanes x 4 elements: lines 4q .. 4q + 3, 16 rows -> each lane its row's four); floats: 32 lines, 64-byte
//                    group c at c ^ (k / 4 % 4), read one by one
// Lines beyond the operand are clamped to its last one (their results are not stored), what lies beyond k reads as zero (an offset beyond
// num_records).
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
#define AIPT_LDS __attribute__((address_space(3)))

// The accumulators are pinned to accumulation registers in place: with the builtin the compiler keeps a part of 64 of them in vector
// registers and moves it to and fro each step (0.84 PFLOP/s of 1.2).  settle() stands between these instructions and everything else that
// touches an accumulator: the compiler does not know that they are matrix instructions, whose results and sources want wait states.
// float: 16 bytes are four k, one for each of four instructions (any order is a sum).
template <typename T> struct Frag;
template <> struct Frag<bf16> {
    using V = bf16x8;
    static constexpr int Q = 1;
    template <int> static __device__ inline void mac(V a, V b, f32x4& c) { asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b)); }
};
template <> struct Frag<f16> {
    using V = f16x8;
    static constexpr int Q = 1;
    template <int> static __device__ inline void mac(V a, V b, f32x4& c) { asm("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b)); }
};
template <> struct Frag<float> {
    using V = f32x4;
    static constexpr int Q = 4;
    // (the next of the four adds to what the last but FJ wrote: with FJ = 2, one instruction of 8 passes lies between, and wait states make it sure)
    template <int q> static __device__ inline void mac(V a, V b, f32x4& c) { asm("s_nop 3\n\tv_mfma_f32_16x16x4_f32 %0, %1, %2, %0" : "+a"(c) : "v"(a[q]), "v"(b[q])); }
};
template <int N> __device__ inline void settle(f32x4* acc) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (i == 0) asm volatile("s_nop 15\n\ts_nop 15" : "+a"(acc[i]));
        else asm volatile("" : "+a"(acc[i]));
    }
}

// loads of one operand's part of a pair: R rows x 128 bytes of k, split over NT threads, W bytes (16, or 4 for lines on 4) a lane
template <int ES, bool KC, int R, int NT, int W> struct TileLoad {
    static constexpr int E = 16 / ES, U = W / ES, KP = 128 / ES, L = R * 128 / (NT * W), GC = ES == 2 ? 2 : 4;   // GC: chunks of a group that stay together
    unsigned off[L];
    int kof[L];                      // the k of this lane's elements within a pair
    const char* base;
    long long step;                  // bytes to the next pair
    __device__ inline void init(const void* p, long long stride, int r0, int rows, int k0, int tid) {
        // (a line's contiguous rows come in whole loads: rows is a multiple of U, or its lines are padded to one)
        base = (const char*)p + (KC ? ((long long)r0 * stride + k0) * ES : ((long long)k0 * stride + r0) * ES);
        step = KC ? 128 : 128 * stride;
        const int last = KC ? rows - 1 - r0 : (rows + U - 1) / U * U - U - r0;
#pragma unroll
        for (int i = 0; i < L; i++) {
            const int at = (i * NT + tid) * W, q = at >> 4, in = (at & 15) / ES;      // chunk, and the element of it
            if (KC) {
                const int r = q >> 3, c = (q & 7) ^ ((r >> 1) & 7);
                off[i] = (unsigned)min(r, last) * (unsigned)(stride * ES) + (c * E + in) * ES;
                kof[i] = c * E + in;
            } else {
                const int k = q / (R / E), c = q % (R / E);
                const int mn = ((c / GC ^ swap(k)) * GC + c % GC) * E + in;
                off[i] = (unsigned)k * (unsigned)(stride * ES) + (unsigned)min(mn, last) * ES;
                kof[i] = k;
            }
        }
    }
    // Which group of line k lies where.  16 bits: the eight lines that 32 lanes read together (k = 0 .. 3, 8 .. 11) begin at as many of the
    // eight 32-byte places of all banks; where lines are shorter than those, by their own places too.  Floats: the four lines of a wave's 64 lanes.
    static __device__ inline int swap(int k) {
        if (ES == 4) return (k >> 2) & (R / 16 < 4 ? R / 16 - 1 : 3);
        if (R == 64) return ((k >> 1) & 1) | ((k >> 2) & 2);
        if (R == 32) return (k >> 3) & 1;
        return (k & 3) | ((k >> 1) & 4);
    }
    // where pair t lies, as a buffer (raw, 2 GiB - 1); load i of it, `left` of k being left.  In assembly: the compiler waits for every load to LDS
    // before a transposing read (vmcnt(0)), and so for loads that are meant for later pairs; the waits are at the barriers.
    __device__ inline i32x4 at(int t) const {
        const unsigned long long p = (unsigned long long)(base + t * step);
        return i32x4{__builtin_amdgcn_readfirstlane((int)p), __builtin_amdgcn_readfirstlane((int)(p >> 32) & 0xffff), 0x7fffffff, 0x00027000};
    }
    __device__ inline void one(int i, i32x4 rs, int left, AIPT_LDS char* lds, int wave) const {
        const unsigned o = kof[i] < left ? off[i] : 0x80000000u;
        const unsigned to = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds + (i * NT + wave * 64) * W));
        if constexpr (W == 16) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(o), "s"(rs) : "memory", "m0");
        else asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(to), "v"(o), "s"(rs) : "memory", "m0");
    }
};

// fragments of N x 16 rows from r0 on: the first or the second half of a pair
template <typename T, bool KC, int R, int N> struct TileRead {
    static constexpr int ES = sizeof(T);
    int at[KC ? 1 : N][2];           // k contiguous: of the two halves; else (16 bits) of the two groups of four k
    __device__ inline void init(int r0, int lane) {
        if constexpr (KC) {
            const int r = r0 + (lane & 15);
#pragma unroll
            for (int h = 0; h < 2; h++) at[0][h] = r * 128 + (((h * 4 + (lane >> 4)) ^ ((r >> 1) & 7)) * 16);
        } else {
#pragma unroll
            for (int n = 0; n < N; n++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int k = ES == 2 ? (lane >> 4) * 8 + h * 4 + ((lane & 15) >> 2) : (lane >> 4) * 4;
                    at[n][h] = k * R * ES + (((r0 / 16 + n) ^ TileLoad<ES, false, R, 64, 16>::swap(k)) * 16 * ES) + (ES == 2 ? (lane & 3) * 8 : (lane & 15) * 4);
                }
        }
    }
    template <int H> __device__ inline typename Frag<T>::V one(int n, AIPT_LDS char* lds) const {
        using V = typename Frag<T>::V;
        if constexpr (KC) return *(AIPT_LDS V*)(lds + at[0][H] + n * 2048);
        else if constexpr (ES == 4) {
            V v;
#pragma unroll
            for (int q = 0; q < 4; q++) v[q] = *(AIPT_LDS float*)(lds + at[n][0] + (H * 16 + q) * R * 4);
            return v;
        } else {
            union { i16x4 h[2]; V v; } u;
            u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((AIPT_LDS i16x4*)(lds + at[n][0] + H * 32 * R * 2));
            u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((AIPT_LDS i16x4*)(lds + at[n][1] + H * 32 * R * 2));
            return u.v;
        }
    }
};

// eight neighbours of a row: bias, activation, residual, 16-byte stores
template <typename T, int ACT, bool ANY> __device__ inline void epilogue8(const GemmArgs& g, int i, int j, float* z, const float* bias_j) {
    float b[8];
    if (g.bias_i) {
        const float v = g.bias ? (float)((const T*)g.bias)[i] : 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) b[e] = v;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) b[e] = bias_j[e];
    }
    struct alignas(16) Oct { T v[8]; } q;
    struct __attribute__((packed, aligned(sizeof(T)))) Loose { unsigned w[2 * sizeof(T)]; };
    auto store = [&](T* p) {
        if constexpr (ANY) *(Loose*)p = __builtin_bit_cast(Loose, q);
        else *(Oct*)p = q;
    };
#pragma unroll
    for (int e = 0; e < 8; e++) z[e] += b[e];
    if (g.pre) {
#pragma unroll
        for (int e = 0; e < 8; e++) q.v[e] = (T)z[e];
        store((T*)g.pre + i * g.pi + j);
    }
#pragma unroll
    for (int e = 0; e < 8; e++) z[e] = act_of<T>(z[e], ACT, g.slope);
    if (g.res) {
        const T* p = (const T*)g.res + i * g.ri + j;
        Oct r;
        if constexpr (ANY) r = __builtin_bit_cast(Oct, *(const Loose*)p);
        else r = *(const Oct*)p;
#pragma unroll
        for (int e = 0; e < 8; e++) z[e] += (float)r.v[e];
    }
#pragma unroll
    for (int e = 0; e < 8; e++) q.v[e] = (T)z[e];
    store((T*)g.c + i * g.cs + j);
}

template <int TI, int TJ, int WI, int WJ, int S> constexpr int tile_lds() {       // bytes: the ring, or the slabs that results go through
    const int ring = S % 2 ? S * TI * 128 : S / 2 * (TI + TJ) * 128, slabs = WI * WJ * (TI / WI < 64 ? TI / WI : 64) * (TJ / WJ) * 4;
    return ring > slabs ? ring : slabs;
}
template <typename T, bool AK, bool BK, int TI, int TJ, int WI, int WJ, int S, int W>
__device__ __forceinline__ void tile_of(const GemmArgs& g, const int block, const int total, AIPT_LDS char* lds) {
    constexpr int NT = WI * WJ * 64, WTI = TI / WI, WTJ = TJ / WJ, FI = WTI / 16, FJ = WTJ / 16;
    static_assert(TI == TJ || S % 2 == 0, "an odd ring's slots hold A and B in turn");
    constexpr int SA = TI * 128, SB = TJ * 128;              // bytes of a slot
    constexpr int SLAB = WTI < 64 ? WTI : 64;                // rows of a wave's results that go through LDS at a time
    using V = typename Frag<T>::V;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // workgroups go round the eight XCDs: each XCD takes a run of neighbouring tiles, which share operands in its L2 ...
    const int per = total >> 3, extra = total & 7, x = block & 7;
    int job = (x < extra ? x * (per + 1) : extra * (per + 1) + (x - extra) * per) + (block >> 3);
    const int tiles = g.tiles_i * g.tiles_j, split = job / tiles;
    job -= split * tiles;
    // ... in columns of 8 tiles
    const int band = 8 * g.tiles_j, b0 = job / band * 8, bh = min(8, g.tiles_i - b0);
    const int i0 = (b0 + (job % band) % bh) * TI, j0 = (job % band) / bh * TJ;
    const int k0 = split * g.k_split, k1 = (int)min((long long)g.K, (long long)k0 + g.k_split), KP = 128 / (int)sizeof(T), n = (k1 - k0 + KP - 1) / KP;

    TileLoad<sizeof(T), AK, TI, NT, W> la;
    TileLoad<sizeof(T), BK, TJ, NT, W> lb;
    la.init(g.a, g.as, i0, g.I, k0, tid);
    lb.init(g.b, g.bs, j0, g.J, k0, tid);
    const int wi = wave / WJ * WTI, wj = wave % WJ * WTJ;
    TileRead<T, AK, TI, FI> ra;
    TileRead<T, BK, TJ, FJ> rb;
    ra.init(wi, lane);
    rb.init(wj, lane);
    constexpr int LA = decltype(la)::L, LB = decltype(lb)::L;
    // bytes from the ring's start to the slot of load u (2 P: A, 2 P + 1: B of pair P); `slot`: u % S
    auto place = [&](int slot) { return lds + (S % 2 ? slot * SA : (slot >> 1) * (SA + SB) + (slot & 1) * SA); };
    auto next = [](int slot, int by) { slot += by; return slot >= S ? slot - S : slot; };
    f32x4 acc[FI][FJ] = {};
    settle<FI * FJ>(&acc[0][0]);
    V a0[FI], b0f[FJ], a1[FI], b1f[FJ];
#pragma unroll
    for (int u = 0; u < S - 1; u++) {
        const int t = u / 2, left = k1 - k0 - t * KP;
        if (u % 2 == 0) {
            const auto rs = la.at(t);
#pragma unroll
            for (int i = 0; i < LA; i++) la.one(i, rs, left, place(u), wave);
        } else {
            const auto rs = lb.at(t);
#pragma unroll
            for (int i = 0; i < LB; i++) lb.one(i, rs, left, place(u), wave);
        }
    }
    // loads behind A(0) B(0), and, at a barrier, behind the pair that it makes visible: they may still be under way
    constexpr int W0 = (S - 3) / 2 * (LA + LB) + (S % 2 ? 0 : LA), W1 = (S - 4) / 2 * (LA + LB) + (S % 2 ? LA : 0);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(W0) : "memory");
#pragma unroll
    for (int p = 0; p < FI; p++) a0[p] = ra.template one<0>(p, place(0));
#pragma unroll
    for (int q = 0; q < FJ; q++) b0f[q] = rb.template one<0>(q, place(1));
    // A step: the products of one half of a pair, from registers, and between them the reads of the next half and the loads of a slot.
    // The order is the program's, not the scheduler's (which would read the next fragments behind the last product, into the registers
    // that these leave, and so wait for them): rows of FJ products, the reads between the first half of the rows, the loads between the
    // second.
    auto step = [&](auto half, auto is_a, int t, AIPT_LDS char* into, AIPT_LDS char* from_a, AIPT_LDS char* from_b, V* a, V* b, V* an, V* bn) {
        constexpr int HALF = decltype(half)::value, LN = decltype(is_a)::value ? LA : LB;
        constexpr int H = FI / 2, R = (FI + FJ + H - 1) / H, G = (LN + H - 1) / H;
        const auto rs = decltype(is_a)::value ? la.at(t) : lb.at(t);
        const int left = k1 - k0 - t * KP;
#pragma unroll
        for (int p = 0; p < FI; p++) {
            if (p < H) {
#pragma unroll
                for (int r = p * R; r < (p + 1) * R && r < FI + FJ; r++) {
                    if (r < FI) an[r] = ra.template one<HALF>(r, from_a);
                    else bn[r - FI] = rb.template one<HALF>(r - FI, from_b);
                }
            } else {
#pragma unroll
                for (int i = (p - H) * G; i < (p - H + 1) * G && i < LN; i++)
                    if constexpr (decltype(is_a)::value) la.one(i, rs, left, into, wave);
                    else lb.one(i, rs, left, into, wave);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int q = 0; q < FJ; q++) Frag<T>::template mac<0>(b[q], a[p], acc[p][q]);
            if constexpr (Frag<T>::Q == 4) {
#pragma unroll
                for (int q = 0; q < FJ; q++) Frag<T>::template mac<1>(b[q], a[p], acc[p][q]);
#pragma unroll
                for (int q = 0; q < FJ; q++) Frag<T>::template mac<2>(b[q], a[p], acc[p][q]);
#pragma unroll
                for (int q = 0; q < FJ; q++) Frag<T>::template mac<3>(b[q], a[p], acc[p][q]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    using std::integral_constant;
    using First = integral_constant<int, 0>;
    using Second = integral_constant<int, 1>;
    // in the first step of pair P the load 2 P - 1 + S goes out, in the second 2 P + S, into the slots of 2 P - 1 and 2 P
    using OddIsA = integral_constant<bool, S % 2 != 0>;      // what 2 P - 1 + S is
    using EvenIsA = integral_constant<bool, S % 2 == 0>;     // what 2 P + S is
    int slot = 0;                    // of A(P)
    for (int P = 0; P < n; P++) {
        const int sb = next(slot, 1), sa2 = next(slot, 2), sb2 = next(slot, 3);
        step(Second{}, OddIsA{}, P + (S - 1) / 2, place(next(slot, S - 1)), place(slot), place(sb), a0, b0f, a1, b1f);
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(W1) : "memory");
        step(First{}, EvenIsA{}, P + S / 2, place(slot), place(sa2), place(sb2), a1, b1f, a0, b0f);
        slot = sa2;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    settle<FI * FJ>(&acc[0][0]);

    // results: through a slab of LDS of the wave's own (chunk c of row r at c ^ (r % 16)), so that rows are stored in 16-byte pieces
    constexpr int XM = WTJ / 4 < 16 ? WTJ / 4 - 1 : 15;
    AIPT_LDS char* slab = lds + wave * (SLAB * WTJ * 4);
    constexpr int LR = WTJ / 8, RPI = 64 / LR;               // lanes of a row, rows of an instruction
    const int j = j0 + wj + lane % LR * 8;
    const bool whole = j + 8 <= g.J;
    float bias_j[8];
#pragma unroll
    for (int e = 0; e < 8; e++) bias_j[e] = g.bias && !g.bias_i && g.splits == 1 && j + e < g.J ? (float)((const T*)g.bias)[j + e] : 0.f;
    // one by one, neighbouring lanes neighbouring elements
    auto narrow = [&](int s) {
        constexpr int LN = WTJ < 64 ? WTJ : 64, RS = 64 / LN;
#pragma unroll
        for (int h = 0; h < WTJ / LN; h++) {
            const int c = h * LN + lane % LN, jj = j0 + wj + c;
            if (jj >= g.J) continue;
            const float bias = g.bias && !g.bias_i ? (float)((const T*)g.bias)[jj] : 0.f;
            const int r0 = lane / LN, ii = i0 + wi + s * SLAB + r0, end = min(SLAB, g.I - (i0 + wi + s * SLAB));
            T* o = (T*)g.c + (long long)ii * g.cs + jj;
            T* pre = g.pre ? (T*)g.pre + ii * g.pi + jj * g.pj : nullptr;
            const T* res = g.res ? (const T*)g.res + ii * g.ri + jj * g.rj : nullptr;
#pragma unroll 4
            for (int r = r0; r < end; r += RS, o += RS * g.cs) {
                float z = *(AIPT_LDS float*)(slab + r * (WTJ * 4) + (((c >> 2) ^ (r & XM)) * 16) + (c & 3) * 4);
                z += g.bias && g.bias_i ? (float)((const T*)g.bias)[ii - r0 + r] : bias;
                if (pre) { *pre = (T)z; pre += RS * g.pi; }
                z = act_of<T>(z, g.act, g.slope);
                if (res) { z += (float)*res; res += RS * g.ri; }
                *o = (T)z;
            }
        }
    };
#pragma unroll
    for (int s = 0; s < WTI / SLAB; s++) {
#pragma unroll
        for (int p = 0; p < SLAB / 16; p++)
#pragma unroll
            for (int q = 0; q < FJ; q++) {
                const int r = p * 16 + (lane & 15), c = q * 4 + (lane >> 4);
                *(AIPT_LDS f32x4*)(slab + r * (WTJ * 4) + ((c ^ (r & XM)) * 16)) = acc[s * (SLAB / 16) + p][q];
            }
        auto rows_by = [&](auto anywhere, int je, auto done) {
            for (int r = lane / LR; r < SLAB; r += RPI) {
                const int i = i0 + wi + s * SLAB + r;
                if (i >= g.I || j >= g.J) continue;
                alignas(16) float z[8];
                const int c = lane % LR * 2;
                *(f32x4*)z = *(AIPT_LDS f32x4*)(slab + r * (WTJ * 4) + ((c ^ (r & XM)) * 16));
                *(f32x4*)(z + 4) = *(AIPT_LDS f32x4*)(slab + r * (WTJ * 4) + (((c + 1) ^ (r & XM)) * 16));
                if constexpr (decltype(anywhere)::value) {
                    if (je != j) {
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const int k = je - (j0 + wj) + e;
                            z[e] = *(AIPT_LDS float*)(slab + r * (WTJ * 4) + (((k >> 2) ^ (r & XM)) * 16) + (k & 3) * 4);
                        }
                    }
                }
                done(i, z);
            }
        };
        auto rows = [&](auto done) { rows_by(integral_constant<bool, false>{}, j, done); };
        if (g.splits > 1) rows([&](int i, float* z) {
            float* o = g.partial + ((long long)split * g.I + i) * g.J + j;
            if (j + 8 <= g.J && !(g.J & 3)) { *(f32x4*)o = *(f32x4*)z; *(f32x4*)(o + 4) = *(f32x4*)(z + 4); }
            else {
#pragma unroll
                for (int e = 0; e < 8; e++) if (j + e < g.J) o[e] = z[e];
            }
        });
        else if (g.cv == 1 || (g.cv == 9 && g.J - (j0 + wj) < 8)) narrow(s);
        else if (g.cv == 8 && !whole) rows([&](int i, float* z) {
#pragma unroll
            for (int e = 0; e < 8; e++) if (j + e < g.J) epilogue<T>(g, i, j + e, z[e]);
        });
        else if (g.cv == 8) {
            if (g.act == AIPT_ACT_NONE) rows([&](int i, float* z) { epilogue8<T, AIPT_ACT_NONE, false>(g, i, j, z, bias_j); });
            else if (g.act == AIPT_ACT_LEAKY) rows([&](int i, float* z) { epilogue8<T, AIPT_ACT_LEAKY, false>(g, i, j, z, bias_j); });
            else if (g.act == AIPT_ACT_SILU) rows([&](int i, float* z) { epilogue8<T, AIPT_ACT_SILU, false>(g, i, j, z, bias_j); });
            else rows([&](int i, float* z) { epilogue8<T, AIPT_ACT_GELU, false>(g, i, j, z, bias_j); });
        } else {                     // rows that begin anywhere: a row's last eight end with it, and some of them are the neighbouring lane's as well (the same bits)
            const int je = whole ? j : g.J - 8;
#pragma unroll
            for (int e = 0; e < 8; e++) bias_j[e] = g.bias && !g.bias_i ? (float)((const T*)g.bias)[je + e] : 0.f;
            auto rows_any = [&](auto done) { rows_by(integral_constant<bool, true>{}, je, done); };
            if (g.act == AIPT_ACT_NONE) rows_any([&](int i, float* z) { epilogue8<T, AIPT_ACT_NONE, true>(g, i, je, z, bias_j); });
            else if (g.act == AIPT_ACT_LEAKY) rows_any([&](int i, float* z) { epilogue8<T, AIPT_ACT_LEAKY, true>(g, i, je, z, bias_j); });
            else if (g.act == AIPT_ACT_SILU) rows_any([&](int i, float* z) { epilogue8<T, AIPT_ACT_SILU, true>(g, i, je, z, bias_j); });
            else rows_any([&](int i, float* z) { epilogue8<T, AIPT_ACT_GELU, true>(g, i, je, z, bias_j); });
        }
    }
}

template <typename T, bool AK, bool BK, int TI, int TJ, int WI, int WJ, int S, int W>
__global__ __launch_bounds__(WI * WJ * 64, 1) void gemm_tile(const GemmArgs g) {
    __shared__ __attribute__((aligned(1024))) char lds[tile_lds<TI, TJ, WI, WJ, S>()];
    tile_of<T, AK, BK, TI, TJ, WI, WJ, S, W>(g, blockIdx.x, gridDim.x, (AIPT_LDS char*)lds);
}
// Both gradients of a small layer in one launch, by tiles of 64 x 64: neither fills the chip.  AK, BK: of the first (nx workgroups); AK2, BK2.
template <typename T, bool AK, bool BK, bool AK2, bool BK2>
__global__ __launch_bounds__(256, 1) void gemm_both(const GemmArgs dx, const GemmArgs dw, const unsigned nx) {
    __shared__ __attribute__((aligned(1024))) char lds[tile_lds<64, 64, 2, 2, 6>()];
    if (blockIdx.x < nx) tile_of<T, AK, BK, 64, 64, 2, 2, 6, 16>(dx, blockIdx.x, nx, (AIPT_LDS char*)lds);
    else tile_of<T, AK2, BK2, 64, 64, 2, 2, 6, 16>(dw, blockIdx.x - nx, gridDim.x - nx, (AIPT_LDS char*)lds);
}

// The splits of a long contraction, added in a fixed order, and the epilogue: four neighbours a thread.  SIDE threads share a result's splits
// (many splits of a small result: one thread for each result ran for 245 us at 368 splits of 64 x 46).
template <typename T, int SIDE> __device__ inline void join(const GemmArgs& g, long long block, long long blocks, float4 (*lds)[16]) {
    constexpr int QUADS = 256 / SIDE;
    const int per = (g.J + 3) / 4, x = threadIdx.x % QUADS, side = threadIdx.x / QUADS;
    const long long quads = (long long)g.I * per, n = (long long)g.I * g.J;
    const bool quad16 = !(g.J & 3);
    for (long long q0 = block * QUADS; q0 < quads; q0 += blocks * QUADS) {
        const long long at = q0 + x;
        const int i = (int)(at / per), j = (int)(at - (long long)i * per) * 4;
        float s[4] = {};
        if (at < quads) {
            const float* p = g.partial + (long long)i * g.J + j;
            if (quad16) {
#pragma unroll 4
                for (int k = side; k < g.splits; k += SIDE) {
                    const float4 v = *(const float4*)(p + k * n);
                    s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
                }
            } else {
#pragma unroll 4
                for (int k = side; k < g.splits; k += SIDE)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[e] += p[k * n + (j + e < g.J ? e : 0)];        // (beyond the line: not stored)
            }
        }
        if constexpr (SIDE > 1) {
            __syncthreads();
            lds[side][x] = make_float4(s[0], s[1], s[2], s[3]);
            __syncthreads();
            if (side) continue;
            s[0] = s[1] = s[2] = s[3] = 0;
#pragma unroll
            for (int k = 0; k < SIDE; k++) {
                const float4 v = lds[k][x];
                s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
            }
        }
        if (at < quads) {
#pragma unroll
            for (int e = 0; e < 4; e++) if (j + e < g.J) epilogue<T>(g, i, j + e, s[e]);
        }
    }
}

constexpr int JOIN_SIDE = 16;
static bool join_by_side(const GemmArgs& g) { return g.splits > 8; }
static size_t join_blocks(const GemmArgs& g) {
    const size_t quads = (size_t)g.I * ((g.J + 3) / 4);
    return join_by_side(g) ? std::min<size_t>((quads + 15) / 16, 8192) : std::min<size_t>((quads + 255) / 256, 4096);
}
template <typename T, int SIDE>
__global__ __launch_bounds__(256) void gemm_join(const GemmArgs g) {
    __shared__ float4 lds[SIDE > 1 ? SIDE : 1][16];
    join<T, SIDE>(g, blockIdx.x, gridDim.x, lds);
}

// ---- a few rows (at most 8): every line of the many is read once, 16 bytes a lane, by the wave that its results belong to: no tile, no split, one
// launch (one row, 2048 x 2048 bf16: 3.7 us; memory would take 1.7).  R lines a wave (their loads are under way together), M rows; the rows stay in the first-level cache.
template <typename T, int M, int R>
__global__ __launch_bounds__(256) void gemm_rows(const GemmArgs g) {
    constexpr int E = 16 / sizeof(T);
    const int lane = threadIdx.x & 63, j0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * R;
    if (j0 >= g.J) return;
    float acc[M][R] = {};
    const T* b[R];
#pragma unroll
    for (int r = 0; r < R; r++) b[r] = (const T*)g.b + (long long)min(j0 + r, g.J - 1) * g.bs;
#pragma unroll 4
    for (int k = lane * E; k < g.K; k += 64 * E) {
        Chunk<T> w[R];
#pragma unroll
        for (int r = 0; r < R; r++) w[r] = *(const Chunk<T>*)(b[r] + k);
#pragma unroll
        for (int m = 0; m < M; m++) {
            const Chunk<T> x = *(const Chunk<T>*)((const T*)g.a + (long long)min(m, g.I - 1) * g.as + k);
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int e = 0; e < E; e++) acc[m][r] = fmaf((float)x.v[e], (float)w[r].v[e], acc[m][r]);
        }
    }
    float mine = 0;                  // lane m R + r: row m, line r
#pragma unroll
    for (int m = 0; m < M; m++)
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float z = wave_sum(acc[m][r]);
            if (lane == m * R + r) mine = z;
        }
    const int m = lane / R, j = j0 + lane % R;
    if (m >= M || m >= g.I || j >= g.J) return;
    if (g.turned) epilogue<T>(g, j, m, mine);
    else epilogue<T>(g, m, j, mine);
}

// ---- lines that begin anywhere (of halves: an element is one or two), copied to lines on 16 bytes, padded with zeros: twice the operand's bytes, once, for loads of 16 bytes
// in every tile that reads it (1375 x 909 by 303 x 909 fp16: 58 us by gemm_any, copy and tiles 5 + 9).  2.6 TB/s, reads and writes.
struct PackArgs {
    struct Lines { const unsigned short* p; Chunk<unsigned short>* to; long long stride, chunks; int len, line; } m[4];      // line: chunks of a line
    int n;
    long long chunks() const { return m[0].chunks + m[1].chunks + m[2].chunks + m[3].chunks; }
    size_t blocks() const { return (size_t)std::min<long long>((chunks() + 255) / 256, 8192); }
};
__device__ inline void pack(const PackArgs& g, long long block, long long blocks) {
    for (int o = 0; o < g.n; o++) {
        const auto& m = g.m[o];
        for (long long c = block * 256 + threadIdx.x; c < m.chunks; c += blocks * 256) {
            const long long l = c / m.line;
            const int k = (int)(c - l * m.line) * 8;
            const unsigned short* s = m.p + l * m.stride + k;
            Chunk<unsigned short> q;
            if (k + 8 <= m.len) {                            // 16 bytes from anywhere: the chip loads them so
                struct __attribute__((packed, aligned(2))) Any { unsigned v[4]; };
                q = __builtin_bit_cast(Chunk<unsigned short>, *(const Any*)s);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) q.v[e] = k + e < m.len ? s[e] : (unsigned short)0;
            }
            m.to[c] = q;
        }
    }
}
__global__ __launch_bounds__(256) void pack_lines(const PackArgs g) { pack(g, blockIdx.x, gridDim.x); }

// ---- dz = dy * act'(z), rounded to the element type (what the products' matrix instructions take; kept in two halves, a high and a low one, it would cost
// both products twice their 122 us at 4096^3, for errors of 1.7e-3 instead of 2.4e-3, root mean square), and its sums over rows, unrounded: dy is read once for both.  V elements a lane: 16 bytes where lines
// lie on 16 bytes, two where they lie on two, else one.  A workgroup takes `high` rows; `across` lanes (a power of two) share a row, so that narrow rows too fill a
// wave, and a lane's columns stay its own.  Memory bounds it (4096 x 4096 bf16 22 us, 4.6 TB/s).  Where rows are the contiguous axis (TURNED): 64 lines (columns) of `high` rows, a wave each.
struct DzArgs {
    const void *dy, *z;
    void* dz;
    float* part;                     // [ceil(M / high)][N] sums over a workgroup's rows, or NULL
    void* sum;                       // ... or, where one workgroup has all rows, the sums themselves
    long long dys, zi, zj, dzs;      // strides from line to line, and both of z's, which may lie the other way
    int M, N;                        // rows and columns of dy
    int line;                        // dz's lines, with their padding (of zeros)
    int high, tiles_n, across, act;
    float slope;
    unsigned blocks;
};
template <typename T, int V, bool TURNED>
__global__ __launch_bounds__(256) void act_backward(const DzArgs g, const PackArgs copies) {
    struct alignas(V * sizeof(T)) E { T v[V]; };
    __shared__ float lds[TURNED ? 1 : 256 * V];
    if (blockIdx.x >= g.blocks) return pack(copies, blockIdx.x - g.blocks, gridDim.x - g.blocks);      // the products' operands that are copied, in the same launch
    const int tm = (int)(blockIdx.x / g.tiles_n), tn = (int)(blockIdx.x % g.tiles_n);
    // V elements: in [is there an element], out [is there one of dz, padding included]
    auto one = [&](const T* dyp, const T* zp, T* dzp, bool in, bool out, float* d) {
        if (in) {
            const E dy = *(const E*)dyp;
#pragma unroll
            for (int i = 0; i < V; i++) d[i] = (float)dy.v[i];
            if (g.act != AIPT_ACT_NONE) {
                const E z = *(const E*)zp;
#pragma unroll
                for (int i = 0; i < V; i++) d[i] *= act_slope_of<T>((float)z.v[i], g.act, g.slope);
            }
        }
        if (out) {
            E o;
#pragma unroll
            for (int i = 0; i < V; i++) o.v[i] = (T)d[i];
            *(E*)dzp = o;
        }
    };
    if constexpr (TURNED) {
        const int lane = threadIdx.x & 63, l1 = min(g.N, tn * 64 + 64), c0 = tm * g.high, c1 = (int)min((long long)max(g.M, g.line), (long long)c0 + g.high);
        for (int l = tn * 64 + (threadIdx.x >> 6); l < l1; l += 4) {
            const T* dyp = (const T*)g.dy + l * g.dys;
            const T* zp = (const T*)g.z + l * g.zj;
            T* dzp = (T*)g.dz + l * g.dzs;
            float along = 0;
#pragma unroll 2
            for (int c = c0 + lane * V; c < c1; c += 64 * V) {
                float d[V] = {};
                one(dyp + c, zp + c * g.zi, dzp + c, c < g.M, g.dz && c < g.line, d);
#pragma unroll
                for (int i = 0; i < V; i++) along += d[i];
            }
            if (g.part || g.sum) {
                along = wave_sum(along);
                if (lane == 0) {
                    if (g.sum) ((T*)g.sum)[l] = (T)along;
                    else g.part[(long long)tm * g.N + l] = along;
                }
            }
        }
    } else {
        const int x = threadIdx.x % g.across, y = threadIdx.x / g.across, down = 256 / g.across;
        int l0 = tm * g.high + y;
        const int c = (tn * g.across + x) * V, l1 = (int)min((long long)g.M, (tm + 1ll) * g.high);
        float sum[V] = {};
        if (c < max(g.N, g.line)) {
            const T* dyp = (const T*)g.dy + l0 * g.dys + c;
            const T* zp = (const T*)g.z + l0 * g.zi + c * g.zj;
            T* dzp = (T*)g.dz + l0 * g.dzs + c;
            const long long dyd = down * g.dys, zd = down * g.zi, dzd = down * g.dzs;
            const bool in = c < g.N, out = g.dz && c < g.line;
            // U rows' loads before the first one's result (which might, for all the compiler knows, be what the next row reads); the last rows one by one
            constexpr int U = V * sizeof(T) == 16 ? 2 : 4;
            auto rows = [&](auto uv, int end) {
                constexpr int UU = decltype(uv)::value;
                for (; l0 + (UU - 1) * down < end; l0 += UU * down) {
                    E dy[UU] = {}, z[UU] = {};
                    if (in) {
#pragma unroll
                        for (int u = 0; u < UU; u++) dy[u] = *(const E*)(dyp + u * dyd);
                        if (g.act != AIPT_ACT_NONE) {
#pragma unroll
                            for (int u = 0; u < UU; u++) z[u] = *(const E*)(zp + u * zd);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < UU; u++) {
                        E o;
#pragma unroll
                        for (int i = 0; i < V; i++) {
                            float d = (float)dy[u].v[i];
                            if (g.act != AIPT_ACT_NONE) d *= act_slope_of<T>((float)z[u].v[i], g.act, g.slope);
                            sum[i] += d;
                            o.v[i] = (T)d;
                        }
                        if (out) *(E*)(dzp + u * dzd) = o;
                    }
                    dyp += UU * dyd; zp += UU * zd; dzp += UU * dzd;
                }
            };
            rows(std::integral_constant<int, U>{}, l1);
            rows(std::integral_constant<int, 1>{}, l1);
        }
        if (!g.part && !g.sum) return;
#pragma unroll
        for (int i = 0; i < V; i++) lds[(y * g.across + x) * V + i] = sum[i];
        __syncthreads();
        for (int k = threadIdx.x; k < g.across * V; k += 256) {
            const int n = tn * g.across * V + k;
            if (n >= g.N) continue;
            float s = 0;
            for (int d = 0; d < down; d++) s += lds[d * g.across * V + k];
            if (g.sum) ((T*)g.sum)[n] = (T)s;
            else g.part[(long long)tm * g.N + n] = s;
        }
    }
}
struct SumArgs {
    const float* part;
    void* out;
    int parts, N;
};
// What is left when both products are done, in one launch: their splits joined and the bias's partial sums added (16 columns x 16 lanes of parts).
template <typename T>
__global__ __launch_bounds__(256) void grad_end(const GemmArgs dx, const GemmArgs dw, const SumArgs g, const unsigned nx, const unsigned nw) {
    __shared__ float4 lds[JOIN_SIDE][16];
    unsigned block = blockIdx.x;
    if (block < nx + nw) {
        const GemmArgs& j = block < nx ? dx : dw;
        const unsigned at = block < nx ? block : block - nx, n = block < nx ? nx : nw;
        if (j.splits > 8) join<T, JOIN_SIDE>(j, at, n, lds);
        else join<T, 1>(j, at, n, lds);
        return;
    }
    float (*sums)[16] = (float (*)[16])lds;
    const int x = threadIdx.x & 15, w = threadIdx.x >> 4, n = (block - nx - nw) * 16 + x;
    float s = 0;
    if (n < g.N) {
#pragma unroll 8
        for (int p = w; p < g.parts; p += 16) s += g.part[(long long)p * g.N + n];
    }
    sums[w][x] = s;
    __syncthreads();
    if (w || n >= g.N) return;
    s = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) s += sums[i][x];
    ((T*)g.out)[n] = (T)s;
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
    if (out && n0 && n1) {           // (elements that are none do not coincide)
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

static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

struct Plan {                        // a product as it will be launched, and the workspace it wants
    GemmArgs g = {};
    bool ak = true, bk = true;
    int tile = 0;                    // 0: gemm_any; -1: gemm_rows; else gemm_tile of this size
    bool small = false;              // ... with loads of 4 bytes
    int rows = 0;                    // of gemm_rows
    PackArgs pack = {};              // operands that are copied first
    size_t pack_bytes = 0, partial_bytes = 0, blocks = 0;
    bool fits = true;
    size_t bytes() const { return pack_bytes + partial_bytes; }
};

// The sizes of gemm_tile, and what they cost: `start` microseconds for a workgroup's first loads and its results, pair[c] for a pair of its steps
// while c + 1 workgroups share the CU, of 16-bit types and of floats (whose matrix instructions bind).  Measured, bf16, where each wins:
// 4096^3: 256 x 256 112 us, 128 x 128 120; 2048^3: 128 x 128 24, 64 x 64 30, 256 x 256 42; 1024^3: 64 x 64 8.0, 128 x 128 12; 942080 x 32 x 64:
// 256 x 32 38, 64 x 64 59, 128 x 128 82; 942080 x 64 x 128: 256 x 64 86, 64 x 64 95, 128 x 128 99.  Floats, 2048^3: 256 x 32 137, 64 x 64 139,
// 128 x 128 137; 942080 x 32 x 64: 256 x 32 89, 256 x 64 116, 64 x 64 121.
static const struct Tile { int i, j, fit; double start, pair[2][3]; } TILES[] = {
    {},
    {256, 256, 1, 12, {{1.4, 0, 0}, {8.0, 0, 0}}},
    {128, 128, 2, 4.5, {{0.6, 1.0, 0}, {2.1, 3.7, 0}}},
    {64, 64, 3, 2.5, {{0.26, 0.36, 0.55}, {0.7, 1.1, 1.4}}},
    {256, 64, 2, 5.5, {{0.8, 1.2, 0}, {2.1, 3.8, 0}}},
    {256, 32, 2, 4, {{0.7, 0.9, 0}, {1.1, 2.0, 0}}},
};
constexpr int NTILES = 6, CUS = 256;

// The tile and how often the contraction is split, by the estimate above: rounds of workgroups, and for a split the partial sums' way out and
// back (a join's launch and some 3.5 TB/s).  small: the lines are on 4 bytes only, whose loads cost the steps half again (floats: a quarter).
static double pick(bool wide, bool small, long long I, long long J, long long pairs, int& tile, long long& splits) {
    double best = 1e30;
    for (int t = 1; t < NTILES; t++) {
        const Tile& c = TILES[t];
        if (small && t != 3 && t != 5) continue;
        const long long tiles = ((I + c.i - 1) / c.i) * ((J + c.j - 1) / c.j);
        for (int fill = 0; fill <= c.fit; fill++) {
            long long s = fill ? std::min(CUS * fill / std::max(1ll, tiles), pairs / 2) : 1;
            if (s < 1 || (fill && s == 1)) continue;
            const long long n = (pairs + s - 1) / s, blocks = tiles * s, full = blocks / (CUS * c.fit), rest = blocks - full * CUS * c.fit;
            auto round = [&](int with) { return c.start + n * c.pair[wide][with - 1] * (small ? wide ? 1.25 : 1.45 : 1); };
            double us = full * round(c.fit);
            if (rest) us += round((int)((rest + CUS - 1) / CUS));
            if (s > 1) us += 4 + (double)(s + 1) * I * J * 4 / 3.5e6;
            if (us < best) { best = us; tile = t; splits = s; }
        }
    }
    return best;
}

// C[i][j] = sum_k A[i][k] B[j][k]; A (I x K) and B (J x K) by their strides; the result's j axis contiguous.  copy_us: what a launch for copies costs
static Plan plan_gemm(int type, View a, View b, long long I, long long J, long long K, double copy_us) {
    Plan p;
    const int es = type_bytes(type), E = 16 / es, ks = 8 * E;
    p.ak = a.second; p.bk = b.second;
    p.g.I = (int)I; p.g.J = (int)J; p.g.K = (int)K;
    // gemm_tile wants lines on 16 bytes that hold whole 16-byte chunks (or, in two of its sizes, on 4), and a tile's lines within 31 bits of
    // its first
    auto unit = [&](const View& v, long long len) {
        if (v.other * es * 256 >= (1ll << 31)) return 0;
        for (int w : {16, 4})
            if (!((uintptr_t)v.p & (w - 1)) && v.other * es % w == 0 && (v.padded || len * es % w == 0)) return w;
        return 0;
    };
    const long long pairs = (K + ks - 1) / ks;
    long long splits = 1;
    int w[2];
    for (int o = 0; o < 2; o++) w[o] = unit(o ? b : a, (o ? b : a).second ? K : o ? J : I);
    // Copied to lines of 16 bytes: 16-bit lines on less than 4; a small operand for whose sake the other would go by 4 too; and whatever lies on 4
    // where the estimate says so, a copy at 2.2 TB/s included (bf16 8192 x 2050 x 2048: 158 -> 92 us; 4096 x 1030 x 1024 27 by loads of 4, 33 copied).
    long long lines[2], line[2];
    bool copy[2];
    for (int o = 0; o < 2; o++) {
        const View& v = o ? b : a;
        const long long rows = o ? J : I;
        line[o] = ((v.second ? K : rows) + E - 1) / E;
        lines[o] = v.second ? rows : K;
        copy[o] = (!w[o] && es == 2) || (w[o] != 16 && w[1 - o] == 16 && lines[o] * line[o] * 16 <= std::max(1ll << 20, (o ? I : J) * K * es / 4));
    }
    if (I && J && (w[0] || copy[0]) && (w[1] || copy[1]) && ((w[0] == 4 && !copy[0]) || (w[1] == 4 && !copy[1]))) {
        double bytes = 0;
        for (int o = 0; o < 2; o++) if (w[o] == 4 && !copy[o]) bytes += (double)lines[o] * line[o] * 16;
        int t = 0;
        if (pick(es == 4, false, I, J, pairs, t, splits) + copy_us + bytes * 2 / 2.2e6 < pick(es == 4, true, I, J, pairs, t, splits))
            for (int o = 0; o < 2; o++) copy[o] |= w[o] == 4;
    }
    for (int o = 0; o < 2; o++) {
        View& v = o ? b : a;
        const long long len = v.second ? K : o ? J : I;
        if (I && J && K && copy[o] && line[o] * 16 * 256 < (1ll << 31)) {
            const int h = es / 2;                            // halves of an element
            p.pack.m[o] = {(const unsigned short*)v.p, (Chunk<unsigned short>*)p.pack_bytes, v.other * h, lines[o] * line[o], (int)len * h, (int)line[o]};   // (`to`: an offset for now)
            p.pack_bytes += up256((size_t)(lines[o] * line[o]) * 16);
            v = {nullptr, v.second ? line[o] * E : 1, v.second ? 1 : line[o] * E, v.second, line[o] * E, true};
            w[o] = 16;
        }
    }
    p.g.a = a.p; p.g.b = b.p;
    p.g.as = a.other; p.g.bs = b.other;
    p.g.avec = !((uintptr_t)a.p & 15) && (a.other % E == 0);
    p.g.bvec = !((uintptr_t)b.p & 15) && (b.other % E == 0);
    splits = 1;
    p.small = std::min(w[0], w[1]) == 4;
    if (w[0] && w[1] && I && J) {
        const double us = pick(es == 4, p.small, I, J, pairs, p.tile, splits);
        // gemm_rows: lines of k on 16 bytes.  3 us and the many lines at 4 TB/s, but no faster than a wave goes along its lines
        const long long few = std::min(I, J), many = std::max(I, J);
        if (p.ak && p.bk && w[0] == 16 && w[1] == 16 && K % E == 0 && !p.pack_bytes && few <= 8 && K &&
            3 + std::max(many * K * es / 4e6, (double)K / (64 * E) * 0.1 * few) < us) {
            p.tile = -1;
            p.g.splits = 1;
            p.g.turned = J < I;
            if (p.g.turned) { std::swap(p.g.a, p.g.b); std::swap(p.g.as, p.g.bs); std::swap(p.g.I, p.g.J); }
            p.rows = few <= 1 ? 1 : few <= 2 ? 2 : few <= 4 ? 4 : 8;
            p.blocks = (size_t)((many + 4 * (p.rows <= 2 ? 2 : 4) - 1) / (4 * (p.rows <= 2 ? 2 : 4)));
            p.fits = grid_fits(p.blocks, 256);
            return p;
        }
    }
    const int ti = p.tile ? TILES[p.tile].i : GT, tj = p.tile ? TILES[p.tile].j : GT, step = ks;
    p.g.tiles_i = (int)((I + ti - 1) / ti); p.g.tiles_j = (int)((J + tj - 1) / tj);
    const long long tiles = (long long)p.g.tiles_i * p.g.tiles_j, steps = pairs;
    // gemm_any: two workgroups a CU, none with fewer than 4 steps
    if (!p.tile) splits = tiles > 0 && tiles < 512 ? std::max(1ll, std::min(512 / tiles, steps / 4)) : 1;
    const long long per = splits > 1 ? (steps + splits - 1) / splits : std::max(1ll, steps);
    splits = std::max(1ll, (steps + per - 1) / per);
    p.g.splits = (int)splits;
    p.g.k_split = (int)std::min<long long>(per * step, 0x7fffffffll - step);
    p.blocks = (size_t)(tiles * splits);
    p.fits = grid_fits(p.blocks, 256);
    if (splits > 1) p.partial_bytes = (size_t)splits * I * J * sizeof(float);
    return p;
}

template <typename T, int TI, int TJ, int WI, int WJ, int S, int W> static void (*tile_kernel(const Plan& p))(GemmArgs) {
    return p.ak ? (p.bk ? gemm_tile<T, true, true, TI, TJ, WI, WJ, S, W> : gemm_tile<T, true, false, TI, TJ, WI, WJ, S, W>)
                : (p.bk ? gemm_tile<T, false, true, TI, TJ, WI, WJ, S, W> : gemm_tile<T, false, false, TI, TJ, WI, WJ, S, W>);
}
template <typename T> static void (*gemm_of(const Plan& p))(GemmArgs) {
    switch (p.tile) {
        case -1: return p.rows == 1 ? gemm_rows<T, 1, 2> : p.rows == 2 ? gemm_rows<T, 2, 2> : p.rows == 4 ? gemm_rows<T, 4, 4> : gemm_rows<T, 8, 4>;
        case 1: return tile_kernel<T, 256, 256, 2, 2, 5, 16>(p);
        case 2: return tile_kernel<T, 128, 128, 2, 2, 5, 16>(p);
        case 3: return p.small ? tile_kernel<T, 64, 64, 2, 2, 6, 4>(p) : tile_kernel<T, 64, 64, 2, 2, 6, 16>(p);
        case 4: return tile_kernel<T, 256, 64, 4, 1, 4, 16>(p);
        case 5: return p.small ? tile_kernel<T, 256, 32, 4, 1, 4, 4>(p) : tile_kernel<T, 256, 32, 4, 1, 4, 16>(p);
    }
    return p.ak ? (p.bk ? gemm_any<T, true, true> : gemm_any<T, true, false>) : (p.bk ? gemm_any<T, false, true> : gemm_any<T, false, false>);
}
// How many elements the epilogue may move together.  A row's last eight may be two lanes', so that a residual in place is not read by eights
// from anywhere.  942080 x 143 fp16: 322 us one by one, 178 by eights; 235520 x 58 bf16 37 by twos, 31; 1375 x 303 fp16 11.1, 9.1.
static int row_unit(int es, const GemmArgs& g) {
    const long long e = 16 / es;
    if ((g.res && g.rj != 1) || (g.pre && g.pj != 1)) return 1;
    if (!(((uintptr_t)g.c | (uintptr_t)g.res | (uintptr_t)g.pre) & 15) && g.cs % e == 0 && (!g.res || g.ri % e == 0) && (!g.pre || g.pi % e == 0)) return 8;
    return g.res == g.c ? 1 : 9;
}

// the product itself, its operands' copies being made: where they lie and the partial sums
static void place(Plan& p, char* ws) {
    for (int o = 0; o < 2; o++) {
        if (!p.pack.m[o].chunks) continue;
        p.pack.m[o].to = (Chunk<unsigned short>*)(ws + (size_t)p.pack.m[o].to);
        (o ? p.g.b : p.g.a) = p.pack.m[o].to;
    }
    p.g.partial = (float*)(ws + p.pack_bytes);
}
template <typename T> static hipError_t launch_gemm(hipStream_t st, Plan& p) {
    p.g.cv = row_unit(sizeof(T), p.g);
    return launch(gemm_of<T>(p), p.blocks, 256, 0, st, p.g);
}
template <typename T> static hipError_t run_gemm_t(hipStream_t st, Plan& p, void* ws) {
    if (!p.blocks) return hipSuccess;
    place(p, (char*)ws);
    hipError_t e = hipSuccess;
    p.pack.n = 2;
    if (p.pack_bytes) e = launch(pack_lines, p.pack.blocks(), 256, 0, st, p.pack);
    if (e == hipSuccess) e = launch_gemm<T>(st, p);
    if (e == hipSuccess && p.g.splits > 1)
        e = join_by_side(p.g) ? launch(gemm_join<T, JOIN_SIDE>, join_blocks(p.g), 256, 0, st, p.g) : launch(gemm_join<T, 1>, join_blocks(p.g), 256, 0, st, p.g);
    return e;
}
static hipError_t run_gemm(int type, hipStream_t st, Plan& p, void* ws) {
    return type == AIPT_TYPE_F32 ? run_gemm_t<float>(st, p, ws) : type == AIPT_TYPE_BF16 ? run_gemm_t<bf16>(st, p, ws) : run_gemm_t<f16>(st, p, ws);
}

// the forward product: turned over (C^T = w x^T) where y's rows are the contiguous axis
static Plan plan_forward(const aipt_linear_args* a) {
    const View x = view_of(a->x, a->m, a->k), w = view_of(a->w, a->n, a->k), y = view_of(a->y, a->m, a->n);
    const bool turn = !y.second;
    Plan p = turn ? plan_gemm(a->type, w, x, a->n, a->m, a->k, 4) : plan_gemm(a->type, x, w, a->m, a->n, a->k, 4);
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
    bool dz_turned = false;
    int dz_v = 1;
    int parts = 0;
    size_t dz_bytes = 0, part_bytes = 0, gemm_bytes = 0, dz_blocks = 0;
    size_t bytes() const { return dz_bytes + part_bytes + gemm_bytes; }
};
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
    if (p.make_dz || p.want_db) {
        DzArgs& g = p.dz;
        const bool turned = !dy.second;
        const long long len = turned ? a->m : a->n, zline = turned ? z.rj : z.ri;
        p.dz_turned = turned;
        p.dz_v = 1;
        for (int v : {2, E}) {
            const bool z_same = a->act == AIPT_ACT_NONE || (z.second == dy.second && !((uintptr_t)z.p & (v * es - 1)) && zline % v == 0);
            if (!((uintptr_t)dy.p & (v * es - 1)) && dy.other % v == 0 && len % v == 0 && z_same) p.dz_v = v;
        }
        const long long wide = std::max<long long>(a->n, turned ? 0 : g.line), v = p.dz_v;
        g.across = 4;
        while (g.across < 256 && g.across * v < wide) g.across *= 2;
        // fewer lanes a row, and more workgroups side by side, where that leaves fewer idle (3431 x 2304 fp16, 288 lanes' worth: 20 us by 256, 15 by 32)
        auto lanes = [&](int across) { return (wide + across * v - 1) / (across * v) * across; };
        for (int across = g.across / 2; across >= 32; across /= 2) if (lanes(across) * 11 < lanes(g.across) * 10) g.across = across;
        g.tiles_n = (int)(turned ? (a->n + 63) / 64 : (wide + g.across * v - 1) / (g.across * v));
        // some 2 048 workgroups, each with 4 rows a thread at least, and no more than 1 024 partial sums a column
        const long long unit = turned ? 64 * v : 256 / g.across, fair = (a->m * g.tiles_n + 2047) / 2048;
        const long long high = std::min((std::max({4 * unit, fair, (a->m + 1023) / 1024}) + unit - 1) / unit * unit, 0x40000000ll);
        const long long tm = (a->m + high - 1) / high;
        g.high = (int)high;
        p.parts = (int)tm;
        if (p.want_db && tm > 1) p.part_bytes = up256((size_t)tm * a->n * sizeof(float));
        g.dy = a->dy.data; g.z = a->preact.data; g.dz = p.make_dz ? d.p : nullptr;
        g.part = p.want_db && tm > 1 ? (float*)(ws + p.dz_bytes) : nullptr;
        g.sum = p.want_db && tm == 1 ? a->dbias : nullptr;
        g.dys = dy.other; g.zi = z.ri; g.zj = z.rj; g.dzs = d.other;
        g.M = (int)a->m; g.N = (int)a->n;
        g.act = a->act; g.slope = a->slope;
        p.dz_blocks = (size_t)tm * g.tiles_n;
    }
    auto flip = [](View v) { std::swap(v.ri, v.rj); v.second = !v.second; return v; };
    if (p.want_dx) {                 // dx[m][k] = sum_n dz[m][n] w[n][k]
        const View w = view_of(a->w, a->n, a->k), o = view_of(a->dx, a->m, a->k);
        p.dx = o.second ? plan_gemm(a->type, d, flip(w), a->m, a->k, a->n, 0) : plan_gemm(a->type, flip(w), d, a->k, a->m, a->n, 0);
        p.dx.g.c = a->dx.data; p.dx.g.cs = o.other;
    }
    if (p.want_dw) {                 // dw[n][k] = sum_m dz[m][n] x[m][k]
        const View x = view_of(a->x, a->m, a->k), o = view_of(a->dw, a->n, a->k);
        p.dw = o.second ? plan_gemm(a->type, flip(d), flip(x), a->n, a->k, a->m, 0) : plan_gemm(a->type, flip(x), flip(d), a->k, a->n, a->m, 0);
        p.dw.g.c = a->dw.data; p.dw.g.cs = o.other;
    }
    p.gemm_bytes = up256(p.want_dx ? p.dx.bytes() : 0) + up256(p.want_dw ? p.dw.bytes() : 0);
    return p;
}

template <typename T> static void (*dz_kernel(const GradPlan& p))(DzArgs, PackArgs) {
    constexpr int V = 16 / sizeof(T);
    if (p.dz_v == V) return p.dz_turned ? act_backward<T, V, true> : act_backward<T, V, false>;
    if (p.dz_v == 2) return p.dz_turned ? act_backward<T, 2, true> : act_backward<T, 2, false>;
    return p.dz_turned ? act_backward<T, 1, true> : act_backward<T, 1, false>;
}

// The gradients: dz with its sums and the operands' copies, the products, and what is left of both -- three to four launches.
template <typename T> static hipError_t run_backward(hipStream_t st, GradPlan& p, const aipt_linear_grad_args* a, char* ws) {
    hipError_t e = hipSuccess;
    PackArgs copies = {};
    char* at = ws + p.dz_bytes + p.part_bytes;
    for (Plan* q : {&p.dx, &p.dw}) {
        if (!q->blocks) continue;
        place(*q, at);
        at += up256(q->bytes());
        for (auto& m : q->pack.m) if (m.chunks) copies.m[copies.n++] = m;
    }
    if (p.dz_blocks) {
        p.dz.blocks = (unsigned)p.dz_blocks;
        e = launch(dz_kernel<T>(p), p.dz_blocks + copies.blocks(), 256, 0, st, p.dz, copies);
    } else if (copies.n) e = launch(pack_lines, copies.blocks(), 256, 0, st, copies);
    if (e == hipSuccess && p.want_db && !a->m) e = zero_fill(st, a->dbias, (size_t)a->n * sizeof(T));
    // where both go by the small tile and the matrices lie all one way: rows, or planar
    const Plan &x = p.dx, &w = p.dw;
    const bool rows = x.ak && !x.bk && !w.ak && !w.bk, planar = !x.ak && x.bk && !w.ak && w.bk;
    if (e == hipSuccess && x.blocks && w.blocks && x.tile == 3 && w.tile == 3 && !x.small && !w.small && (rows || planar) && grid_fits(x.blocks + w.blocks, 256)) {
        p.dx.g.cv = row_unit(sizeof(T), x.g);
        p.dw.g.cv = row_unit(sizeof(T), w.g);
        e = launch(rows ? gemm_both<T, true, false, false, false> : gemm_both<T, false, true, false, true>, x.blocks + w.blocks, 256, 0, st, x.g, w.g, (unsigned)x.blocks);
    } else
        for (Plan* q : {&p.dx, &p.dw}) if (e == hipSuccess && q->blocks) e = launch_gemm<T>(st, *q);
    const size_t nx = p.dx.blocks && p.dx.g.splits > 1 ? join_blocks(p.dx.g) : 0, nw = p.dw.blocks && p.dw.g.splits > 1 ? join_blocks(p.dw.g) : 0,
                 nb = p.want_db && p.parts > 1 ? (size_t)((a->n + 15) / 16) : 0;
    if (e == hipSuccess && nx + nw + nb) e = launch(grad_end<T>, nx + nw + nb, 256, 0, st, p.dx.g, p.dw.g, SumArgs{p.dz.part, a->dbias, p.parts, (int)a->n}, (unsigned)nx, (unsigned)nw);
    return e;
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

static aipt_linear_plan planned(const Plan& p) {
    if (!p.blocks) return {};
    const int copied = (p.pack.m[0].chunks ? 1 : 0) | (p.pack.m[1].chunks ? 2 : 0), lines = (p.ak ? 1 : 0) | (p.bk ? 2 : 0);
    if (p.tile < 0) return {0, p.rows, 16, lines, copied, p.g.splits};
    return {p.tile ? TILES[p.tile].i : GT, p.tile ? TILES[p.tile].j : GT, !p.tile ? 0 : p.small ? 4 : 16, lines, copied, p.g.splits};
}

}  // namespace aipt

using aipt::fail;

extern "C" {

int aipt_linear_workspace(aipt_ctx* ctx, const aipt_linear_args* a, size_t* bytes) {
    if (!bytes) return fail(ctx, AIPT_E_INVALID, "aipt_linear_workspace: bytes is NULL");
    const int rc = aipt::forward_check(ctx, "aipt_linear_workspace", a, false);
    if (rc) return rc;
    *bytes = aipt::plan_forward(a).bytes();
    return AIPT_OK;
}

int aipt_linear_planned(aipt_ctx* ctx, const aipt_linear_args* a, aipt_linear_plan* plan) {
    if (!plan) return fail(ctx, AIPT_E_INVALID, "aipt_linear_planned: plan is NULL");
    const int rc = aipt::forward_check(ctx, "aipt_linear_planned", a, false);
    if (rc) return rc;
    *plan = aipt::planned(aipt::plan_forward(a));
    return AIPT_OK;
}

int aipt_linear(aipt_ctx* ctx, const aipt_linear_args* a, void* d_workspace, size_t workspace_bytes) {
    const char* me = "aipt_linear";
    const int rc = aipt::forward_check(ctx, me, a, true);
    if (rc) return rc;
    const int es = aipt::type_bytes(a->type);
    aipt::Plan p = aipt::plan_forward(a);
    if (!p.fits) return fail(ctx, AIPT_E_INVALID, "%s: %lld x %lld has too many tiles", me, a->m, a->n);
    if (p.bytes() && (!d_workspace || workspace_bytes < p.bytes() || ((uintptr_t)d_workspace & 255)))
        return fail(ctx, AIPT_E_INVALID, "%s: workspace of %zu bytes, %zu are wanted, 256-byte aligned", me, workspace_bytes, p.bytes());
    const aipt::Extent x = aipt::extent_of(a->x, a->m, a->k, es), w = aipt::extent_of(a->w, a->n, a->k, es), y = aipt::extent_of(a->y, a->m, a->n, es),
                       r = aipt::extent_of(a->residual, a->m, a->n, es), z = aipt::extent_of(a->preact, a->m, a->n, es), b = {(const char*)a->bias, 1, a->n * es, 0},
                       s = {(const char*)d_workspace, 1, (long long)p.bytes(), 0};
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

int aipt_linear_backward_planned(aipt_ctx* ctx, const aipt_linear_grad_args* a, aipt_linear_plan* dx, aipt_linear_plan* dw) {
    if (!dx || !dw) return fail(ctx, AIPT_E_INVALID, "aipt_linear_backward_planned: dx or dw is NULL");
    const int rc = aipt::backward_check(ctx, "aipt_linear_backward_planned", a, false);
    if (rc) return rc;
    const aipt::GradPlan p = aipt::plan_backward(a, nullptr);
    *dx = aipt::planned(p.dx);
    *dw = aipt::planned(p.dw);
    return AIPT_OK;
}

int aipt_linear_backward(aipt_ctx* ctx, const aipt_linear_grad_args* a, void* d_workspace, size_t workspace_bytes) {
    const char* me = "aipt_linear_backward";
    const int rc = aipt::backward_check(ctx, me, a, true);
    if (rc) return rc;
    const int es = aipt::type_bytes(a->type);
    aipt::GradPlan p = aipt::plan_backward(a, (char*)d_workspace);
    if ((p.want_dx && !p.dx.fits) || (p.want_dw && !p.dw.fits) || !aipt::grid_fits(p.dz_blocks + 8192, 256))
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
    char* ws = (char*)d_workspace;
    AIPT_HIP(ctx, t == AIPT_TYPE_F32 ? aipt::run_backward<float>(st, p, a, ws) : t == AIPT_TYPE_BF16 ? aipt::run_backward<aipt::bf16>(st, p, a, ws) : aipt::run_backward<aipt::f16>(st, p, a, ws));
    return AIPT_OK;
}

}  // extern "C"
