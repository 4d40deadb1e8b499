// adamw.hip -- one AdamW step over many tensors (aipt_adamw_*).
//
// What it cannot do without: p in and out, the gradient, the state in and out -- 28 bytes a parameter with fp32 state and gradients,
// 14 with 8-bit state and bf16 gradients -- and some 40 operations on them: memory bounds it, and for small sets the launch.  So: ONE
// launch over all tensors, a wave per 256-element block (16-byte accesses, and the block's scale is a wave's own maximum), and the step
// number on the device, advanced by the last workgroup, so that neither the host nor a second launch has a part in it.  The table of tensors
// lies in device memory, read by scalar loads: the kernel arguments of a launch hold a hundred at most.
// Measured: 252 M parameters, 8-bit state, bf16 gradients and copies 890 us (4.5 TB/s; a large copy reaches 5.05); the denoiser's 1.5 M, 32-bit state,
// 10 us and 4 for the norm.
#include "layer_ops.h"

#include <cmath>
#include <new>

namespace aipt {

constexpr int BLOCK = 256;           // elements that share a scale; what one wave handles at a time
constexpr int GRID = 2048;           // most workgroups of a launch: 8 a CU; the blocks beyond 4 a workgroup go round
constexpr int COUNTERS = 32;         // of finished workgroups, a 128-byte line each
constexpr size_t SCRATCH = (COUNTERS + 1) * 128;             // bytes of the workspace before the partial sums
constexpr float TOP = 448.f;         // largest e4m3
constexpr float LIVE = 0x1p-100f;    // blocks below this are kept as zeros (448 / top stays finite)

struct AdamTensor {
    float* p;
    const void* g;
    void* copy;
    long long count;
    unsigned first;                  // its first block
    float decay;
};

// The table is written once, before any launch that reads it, and never by a kernel: constant memory to the compiler, so that a wave's look-ups are scalar.
typedef const __attribute__((address_space(4))) AdamTensor* AdamTable;

struct AdamArgs {
    const AdamTensor* tab;
    int n;
    unsigned blocks;
    void *m, *v;
    float *ms, *vs;
    int* step;
    const double* partial;           // sums of the gradients' squares to clip by, or NULL
    float* norm;                     // receives their root
    int npartial;
    float max_norm;
    unsigned* ticket;                // workgroups done: the last one advances `step`
    double ln1, ln2;                 // logarithms of the betas
    float lr, beta1, beta2, eps;
    float omb1, omb2;                // 1 - beta, rounded once: 1 - 0.999f is 5e-5 off 0.001
    unsigned seed;
    int pad;
};

template <typename G> __device__ inline void load4(const G* g, float* o);
template <> __device__ inline void load4<float>(const float* g, float* o) {
    const float4 q = *(const float4*)g;
    o[0] = q.x; o[1] = q.y; o[2] = q.z; o[3] = q.w;
}
template <> __device__ inline void load4<bf16>(const bf16* g, float* o) {
    struct alignas(8) Q { bf16 v[4]; } q = *(const Q*)g;
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = (float)q.v[i];
}
template <> __device__ inline void load4<f16>(const f16* g, float* o) {
    struct alignas(8) Q { f16 v[4]; } q = *(const Q*)g;
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = (float)q.v[i];
}

// e4m3 <-> float: the chip's own conversions (OCP e4m3 on gfx950; to nearest even, and these values are at most 448)
__device__ inline void from_e4m3(unsigned q, float* o) {
    o[0] = __builtin_amdgcn_cvt_f32_fp8(q, 0);
    o[1] = __builtin_amdgcn_cvt_f32_fp8(q, 1);
    o[2] = __builtin_amdgcn_cvt_f32_fp8(q, 2);
    o[3] = __builtin_amdgcn_cvt_f32_fp8(q, 3);
}
__device__ inline unsigned to_e4m3(const float* o) {
    int q = __builtin_amdgcn_cvt_pk_fp8_f32(o[0], o[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(o[2], o[3], q, true);
}

// x > 0 to one of the two e4m3 values around it, up with the probability of its distance from the lower one: the mean is x.  Steps of 2^-9 below
// 2^-6, of an eighth of the binade above; `random`: 24 of its bits count.  (The chip's own conversion by chance takes 20, truncated; this
// one is the formula in fp32, so that whoever works it out gets the same bits.)
__device__ inline unsigned chance_e4m3(float x, unsigned random) {
    const int e = max(__builtin_amdgcn_frexp_expf(x), -5);                 // x < 2^e
    const float q = __builtin_amdgcn_ldexpf(x, 4 - e) + (float)(random >> 8) * 0x1p-24f;
    return min((unsigned)((e + 5) * 8 + (int)q), 126u);                    // exponent field and mantissa at once, carries included; 126: 448
}

// 32 random bits from a place and a key: multiplications by odd constants (fractions of the golden ratio and of the roots of 3 and 5)
// carry low bits up, the shifts bring high ones down
__device__ inline unsigned hash(unsigned long long place, unsigned key) {
    unsigned x = (unsigned)(place ^ (place >> 32)) ^ key;
    x *= 0x9E3779B1u; x ^= x >> 15;
    x *= 0xBB67AE85u; x ^= x >> 13;
    x *= 0x3C6EF373u;
    return x ^ (x >> 16);
}

// Where block b lies: `ti` its tensor (blocks only grow, so a wave's search goes on from its last one's), `at` the lane's first element,
// the return value how many of the lane's four exist (<= 0: none).
__device__ inline int locate(AdamTable tab, int n, unsigned b, int lane, int& ti, long long& at) {
    int hi = n;
    while (hi - ti > 1) {
        const int mid = (ti + hi) >> 1;
        if (tab[mid].first <= b) ti = mid; else hi = mid;
    }
    at = (long long)(b - tab[ti].first) * BLOCK + lane * 4;
    const long long left = tab[ti].count - at;
    return left > 4 ? 4 : (int)left;
}

// what a wave holds of a block: a lane four elements
template <typename C, int BITS> struct AdamBlock {
    float p[4], g[4], m[4], v[4], ms, vs, decay;
    unsigned mq, vq;
    float* pp;
    C* cp;
    int left;
    bool wide;
};

// The next block's loads are under way while one is worked on; the first one's, while the bias and the clipping are worked out.
template <typename G, typename C, int BITS>
__global__ __launch_bounds__(256) void adamw_step(const AdamArgs a) {
    __shared__ double norms[4];
    const AdamTable tab = (AdamTable)(uintptr_t)a.tab;
    const int lane = threadIdx.x & 63;
    const unsigned waves = gridDim.x * 4;
    int ti = 0;
    using Block = AdamBlock<C, BITS>;
    auto load = [&](unsigned b, Block& q) {
        long long at;
        q.left = locate(tab, a.n, b, lane, ti, at);
        float* const tp = tab[ti].p;
        const void* const tg = tab[ti].g;
        void* const tc = tab[ti].copy;
        q.decay = tab[ti].decay;
        q.pp = tp + at;
        q.cp = tc ? (C*)tc + at : nullptr;
        const G* gp = (const G*)tg + at;
        q.wide = q.left >= 4 && !(((uintptr_t)tp & 15) | ((uintptr_t)tg & (4 * sizeof(G) - 1)) | ((uintptr_t)tc & (4 * sizeof(C) - 1)));
        if (q.wide) {
            load4<float>(q.pp, q.p);
            load4<G>(gp, q.g);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) { q.p[i] = i < q.left ? q.pp[i] : 0.f; q.g[i] = i < q.left ? (float)gp[i] : 0.f; }
        }
        const unsigned long long place = (unsigned long long)b * BLOCK + lane * 4;
        if constexpr (BITS == 32) {
            load4<float>((const float*)a.m + place, q.m);
            load4<float>((const float*)a.v + place, q.v);
        } else {
            q.mq = ((const unsigned*)a.m)[place >> 2];
            q.vq = ((const unsigned*)a.v)[place >> 2];
            q.ms = a.ms[b];
            q.vs = a.vs[b];
        }
    };
    unsigned b = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    Block q;
    if (b < a.blocks) load(b, q);

    const int step = *a.step + 1;
    // 1 - beta^t without the cancellation: lane 0 of beta1, lane 1 of beta2
    const float bias = lane < 2 ? (float)-expm1((double)step * (lane ? a.ln2 : a.ln1)) : 1.f;
    const float rate = a.lr / __shfl(bias, 0), root2 = 1.f / sqrtf(__shfl(bias, 1));
    float factor = 1.f;
    bool skip = false;
    if (a.partial) {                 // every workgroup adds the partial sums, in the same order: cheaper than a launch of its own
        double s = 0;
        for (int i = threadIdx.x; i < a.npartial; i += 256) s += a.partial[i];
#pragma unroll
        for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
        if (lane == 0) norms[threadIdx.x >> 6] = s;
        __syncthreads();
        const float norm = (float)sqrt((norms[0] + norms[1]) + (norms[2] + norms[3]));
        factor = fminf(1.f, a.max_norm / (norm + 1e-6f));
        skip = !(norm <= 3.4028235e38f);                                   // inf and NaN
        if (blockIdx.x == 0 && threadIdx.x == 0) *a.norm = norm;
    }
    const unsigned key = a.seed + (unsigned)step * 0x9E3779B1u;
    if (!skip)
        for (; b < a.blocks; b += waves) {
            Block nq;
            if (b + waves < a.blocks) load(b + waves, nq);
            const unsigned long long place = (unsigned long long)b * BLOCK + lane * 4;
            if constexpr (BITS == 8) {
                from_e4m3(q.mq, q.m);
                from_e4m3(q.vq, q.v);
#pragma unroll
                for (int i = 0; i < 4; i++) { q.m[i] *= q.ms; q.v[i] *= q.vs; q.v[i] *= q.v[i]; }
            }
            const float keep = 1.f - a.lr * q.decay;
            float r[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float gi = q.g[i] * factor;
                q.m[i] = q.m[i] * a.beta1 + gi * a.omb1;
                q.v[i] = q.v[i] * a.beta2 + gi * gi * a.omb2;
                // the chip's root and reciprocal, an ulp each: the step is within 6 ulp of itself, far below the parameter's own (a root that is stored is exact).
                // That root takes no subnormal numbers, which an eps of 0 would be felt by: they are scaled, by powers of two
                const bool tiny = q.v[i] < 0x1p-96f;
                r[i] = BITS == 8 ? sqrtf(q.v[i]) : __builtin_amdgcn_sqrtf(tiny ? q.v[i] * 0x1p64f : q.v[i]) * (tiny ? 0x1p-32f : 1.f);
                q.p[i] = q.p[i] * keep - rate * q.m[i] * __builtin_amdgcn_rcpf(r[i] * root2 + a.eps);
            }
            if (q.wide) {
                *(float4*)q.pp = make_float4(q.p[0], q.p[1], q.p[2], q.p[3]);
                if (q.cp) {
                    struct alignas(4 * sizeof(C)) Q { C v[4]; } c;
#pragma unroll
                    for (int i = 0; i < 4; i++) c.v[i] = (C)q.p[i];
                    *(Q*)q.cp = c;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) if (i < q.left) { q.pp[i] = q.p[i]; if (q.cp) q.cp[i] = (C)q.p[i]; }
            }
            if (q.left < 4) {                                              // the padding is zero and stays so
#pragma unroll
                for (int i = 0; i < 4; i++) if (i >= q.left) q.m[i] = q.v[i] = r[i] = 0;
            }
            if constexpr (BITS == 32) {
                *(float4*)((float*)a.m + place) = make_float4(q.m[0], q.m[1], q.m[2], q.m[3]);
                *(float4*)((float*)a.v + place) = make_float4(q.v[0], q.v[1], q.v[2], q.v[3]);
            } else {
                // (a NaN is the largest, and so the scale: the block's state is spoilt, not plausible; fabsf of the root for the sign of a NaN)
                float mt = 0, vt = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) { mt = max_magnitude(mt, fabsf(q.m[i])); vt = max_magnitude(vt, fabsf(r[i])); }
                mt = wave_max_magnitude(mt);
                vt = wave_max_magnitude(vt);
                const bool ml = !(mt < LIVE), vl = !(vt < LIVE);
                const float mi = ml ? 1.f / mt * TOP : 0.f, vi = vl ? 1.f / vt * TOP : 0.f;
                unsigned vq = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    q.m[i] = fminf(fmaxf(q.m[i] * mi, -TOP), TOP);
                    // what is not zero begins at the least e4m3, so that it stays so
                    const unsigned code = chance_e4m3(fmaxf(r[i] * vi, 0x1p-9f), hash(place + i, key));
                    vq |= (r[i] > 0.f && vl ? code : 0u) << (8 * i);
                }
                ((unsigned*)a.m)[place >> 2] = to_e4m3(q.m);
                ((unsigned*)a.v)[place >> 2] = vq;
                if (lane == 0) {
                    a.ms[b] = ml ? mt * (1.f / TOP) : 0.f;
                    a.vs[b] = vl ? vt * (1.f / TOP) : 0.f;
                }
            }
            q = nq;
        }
    // The last workgroup advances the step number: every wave of a workgroup has read it (and waited for what it read) before the barrier behind which
    // the workgroup counts itself.  Nothing is
    // handed from one to another, so there is no fence: a release writes the L2s back, workgroup by workgroup (50 us here).  One counter
    // for all would take 15 ns a workgroup, one after the other: each counts at one of 32, and the last of those at the last.
    __syncthreads();
    if (threadIdx.x == 0) {
        auto count = [&](int at) { return __hip_atomic_fetch_add(a.ticket + at * 32, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
        const unsigned c = blockIdx.x % COUNTERS, mine = (gridDim.x - c + COUNTERS - 1) / COUNTERS, used = min((unsigned)COUNTERS, gridDim.x);
        if (count((int)c) == mine - 1) {
            a.ticket[c * 32] = 0;
            if (count(COUNTERS) == used - 1) {
                a.ticket[COUNTERS * 32] = 0;
                if (!skip) *a.step = step;
            }
        }
    }
}

// ---- the norm of all gradients: partial sums of squares in fixed places, which the step adds.  It reads the gradients once more than the
// step itself would, and there is no way round it: no parameter may change before the last gradient has been seen.  In fp64, which holds the square of
// every gradient: in fp32 one of 1.9e19 made the norm infinite, and the step was skipped.
struct NormArgs {
    const AdamTensor* tab;
    int n;
    unsigned blocks;
    double* partial;                 // one for each workgroup
};
template <typename G>
__global__ __launch_bounds__(256) void grad_square(const NormArgs a) {
    const AdamTable tab = (AdamTable)(uintptr_t)a.tab;
    const int lane = threadIdx.x & 63;
    const unsigned waves = gridDim.x * 4;
    int ti = 0;
    double s = 0;
    for (unsigned b = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)); b < a.blocks; b += waves) {
        long long at;
        const int left = locate(tab, a.n, b, lane, ti, at);
        const void* const tg = tab[ti].g;
        const G* gp = (const G*)tg + at;
        float g[4] = {};
        if (left >= 4 && !((uintptr_t)tg & (4 * sizeof(G) - 1))) load4<G>(gp, g);
        else {
#pragma unroll
            for (int i = 0; i < 4; i++) if (i < left) g[i] = (float)gp[i];
        }
#pragma unroll
        for (int i = 0; i < 4; i++) s = fma((double)g[i], (double)g[i], s);
    }
    __shared__ double part[4];
#pragma unroll
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if (lane == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.partial[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

}  // namespace aipt

static_assert(sizeof(aipt_adamw_tensor) == 40, "argument record (api.py packs it by field)");

struct aipt_adamw {
    aipt_ctx* ctx = nullptr;
    int grad_type = 0, copy_type = 0, bits = 0;
    aipt::AdamArgs args = {};
    unsigned grid = 0;
    double* partial = nullptr;       // in the caller's workspace
};

namespace aipt {

typedef void (*AdamKernel)(AdamArgs);
typedef void (*NormKernel)(NormArgs);
template <typename G> static AdamKernel adam_of(int copy_type, int bits) {
    if (copy_type == AIPT_TYPE_BF16) return bits == 32 ? adamw_step<G, bf16, 32> : adamw_step<G, bf16, 8>;
    return bits == 32 ? adamw_step<G, f16, 32> : adamw_step<G, f16, 8>;
}

}  // namespace aipt

using aipt::fail;

extern "C" {

long long aipt_adamw_state_elements(const long long* counts, int n) {
    if (n < 0 || (n > 0 && !counts)) return AIPT_E_INVALID;
    long long blocks = 0;
    for (int i = 0; i < n; i++) {
        if (counts[i] < 0 || counts[i] > (1ll << 40)) return AIPT_E_INVALID;
        blocks += (counts[i] + aipt::BLOCK - 1) / aipt::BLOCK;
    }
    return blocks * aipt::BLOCK;
}

long long aipt_adamw_workspace(const long long* counts, int n) {
    if (aipt_adamw_state_elements(counts, n) < 0) return AIPT_E_INVALID;
    return (long long)(aipt::SCRATCH + aipt::GRID * sizeof(double) + (size_t)n * sizeof(aipt::AdamTensor));
}

int aipt_adamw_create(aipt_ctx* ctx, const aipt_adamw_tensor* tensors, int n, int grad_type, int copy_type, int state_bits,
                      void* m, void* v, float* m_scale, float* v_scale, int* step, float* norm, void* d_workspace,
                      size_t workspace_bytes, aipt_adamw** out) {
    if (!out) return fail(ctx, AIPT_E_INVALID, "aipt_adamw_create: out is NULL");
    *out = nullptr;
    if (n < 0 || (n > 0 && !tensors)) return fail(ctx, AIPT_E_INVALID, "aipt_adamw_create: %d tensors", n);
    if (!aipt::type_ok(grad_type)) return fail(ctx, AIPT_E_INVALID, "aipt_adamw_create: grad_type %d", grad_type);
    if (copy_type != AIPT_TYPE_BF16 && copy_type != AIPT_TYPE_F16) return fail(ctx, AIPT_E_INVALID, "aipt_adamw_create: copy_type %d (bf16 or f16)", copy_type);
    if (state_bits != 32 && state_bits != 8) return fail(ctx, AIPT_E_INVALID, "aipt_adamw_create: state_bits %d (32 or 8)", state_bits);
    if (!step || !norm || !d_workspace) return fail(ctx, AIPT_E_INVALID, "aipt_adamw_create: step, norm or d_workspace is NULL");
    long long blocks = 0;
    for (int i = 0; i < n; i++) {
        const aipt_adamw_tensor& t = tensors[i];
        if (t.count < 0 || t.count > (1ll << 40)) return fail(ctx, AIPT_E_INVALID, "aipt_adamw_create: tensor %d has %lld elements", i, t.count);
        if (t.count && (!t.param || !t.grad)) return fail(ctx, AIPT_E_INVALID, "aipt_adamw_create: tensor %d: NULL param or grad", i);
        const size_t ga = aipt::type_bytes(grad_type) - 1;
        if (((uintptr_t)t.param & 3) || ((uintptr_t)t.grad & ga) || ((uintptr_t)t.copy & 1)) return fail(ctx, AIPT_E_INVALID, "aipt_adamw_create: tensor %d: misaligned pointer", i);
        if (!std::isfinite(t.weight_decay)) return fail(ctx, AIPT_E_INVALID, "aipt_adamw_create: tensor %d: weight_decay is not finite", i);
        blocks += (t.count + aipt::BLOCK - 1) / aipt::BLOCK;
    }
    if (blocks && (!m || !v)) return fail(ctx, AIPT_E_INVALID, "aipt_adamw_create: m or v is NULL");
    if (blocks && state_bits == 8 && (!m_scale || !v_scale)) return fail(ctx, AIPT_E_INVALID, "aipt_adamw_create: 8-bit state wants m_scale and v_scale");
    const size_t sa = state_bits == 32 ? 15 : 3;
    if (((uintptr_t)m & sa) || ((uintptr_t)v & sa) || ((uintptr_t)m_scale & 3) || ((uintptr_t)v_scale & 3) || ((uintptr_t)step & 3) || ((uintptr_t)norm & 3) || ((uintptr_t)d_workspace & 15))
        return fail(ctx, AIPT_E_INVALID, "aipt_adamw_create: m and v are aligned to four elements, scales, step and norm to one, d_workspace to 16 bytes");
    // what a step writes may not be what it reads elsewhere: sorted by address, neighbours are apart
    {
        std::vector<aipt::Extent> mem;
        std::vector<int> rank;
        try {
            auto add = [&](const void* q, long long bytes, bool written) { if (q && bytes) { mem.push_back({(const char*)q, 1, bytes, bytes}); rank.push_back(written); } };
            for (int i = 0; i < n; i++) {
                add(tensors[i].param, tensors[i].count * 4, true);
                add(tensors[i].copy, tensors[i].count * 2, true);
                add(tensors[i].grad, tensors[i].count * aipt::type_bytes(grad_type), false);
            }
            const long long el = blocks * aipt::BLOCK, sb = state_bits == 32 ? 4 : 1;
            add(m, el * sb, true); add(v, el * sb, true);
            if (state_bits == 8) { add(m_scale, blocks * 4, true); add(v_scale, blocks * 4, true); }
            add(step, 4, true); add(norm, 4, true); add(d_workspace, (long long)workspace_bytes, true);
            std::vector<size_t> order(mem.size());
            for (size_t i = 0; i < order.size(); i++) order[i] = i;
            std::sort(order.begin(), order.end(), [&](size_t x, size_t y) { return mem[x].data < mem[y].data; });
            const char *end_any = nullptr, *end_written = nullptr;       // furthest end so far, of all and of what is written
            for (size_t i : order) {
                if (mem[i].data < end_written || (rank[i] && mem[i].data < end_any))
                    return fail(ctx, AIPT_E_INVALID, "aipt_adamw_create: memory that a step writes overlaps another tensor's, the state's, step or norm");
                const char* e = mem[i].data + mem[i].len;
                end_any = std::max(end_any, e);
                if (rank[i]) end_written = std::max(end_written, e);
            }
        } catch (const std::bad_alloc&) {
            return fail(ctx, AIPT_E_NOMEM, "aipt_adamw_create: out of host memory");
        }
    }
    if (blocks > 0xffffff00ll) return fail(ctx, AIPT_E_INVALID, "aipt_adamw_create: %lld blocks of 256 elements are too many", blocks);
    const size_t need = aipt::SCRATCH + aipt::GRID * sizeof(double) + (size_t)n * sizeof(aipt::AdamTensor);
    if (workspace_bytes < need) return fail(ctx, AIPT_E_INVALID, "aipt_adamw_create: workspace of %zu bytes, %zu are wanted", workspace_bytes, need);
    AIPT_NEED_CTX(ctx);
    std::vector<aipt::AdamTensor> tab;
    aipt_adamw* a = nullptr;
    try {
        unsigned first = 0;
        for (int i = 0; i < n; i++) {
            const aipt_adamw_tensor& t = tensors[i];
            if (!t.count) continue;
            tab.push_back({t.param, t.grad, t.copy, t.count, first, t.weight_decay});
            first += (unsigned)((t.count + aipt::BLOCK - 1) / aipt::BLOCK);
        }
        a = new aipt_adamw();
    } catch (const std::bad_alloc&) {
        return fail(ctx, AIPT_E_NOMEM, "aipt_adamw_create: out of host memory");
    }
    a->ctx = ctx; a->grad_type = grad_type; a->copy_type = copy_type; a->bits = state_bits;
    a->partial = (double*)((char*)d_workspace + aipt::SCRATCH);
    aipt::AdamTensor* d_tab = (aipt::AdamTensor*)(a->partial + aipt::GRID);
    a->args.tab = d_tab; a->args.n = (int)tab.size(); a->args.blocks = (unsigned)blocks;
    a->args.m = m; a->args.v = v; a->args.ms = m_scale; a->args.vs = v_scale; a->args.step = step; a->args.ticket = (unsigned*)d_workspace; a->args.norm = norm;
    a->grid = (unsigned)std::min<long long>((blocks + 3) / 4, aipt::GRID);
    if (!tab.empty()) {
        aipt::DeviceScope dev(ctx->device);
        hipError_t e = dev.err;
        if (e == hipSuccess) e = hipMemcpyAsync(d_tab, tab.data(), tab.size() * sizeof(tab[0]), hipMemcpyHostToDevice, ctx->stream);
        if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
        if (e != hipSuccess) {
            delete a;
            return fail(ctx, AIPT_E_HIP, "aipt_adamw_create: the table's upload: %s", hipGetErrorString(e));
        }
    }
    *out = a;
    return AIPT_OK;
}

int aipt_adamw_step(aipt_ctx* ctx, aipt_adamw* a, double lr, double beta1, double beta2, double eps, double max_norm, uint32_t seed) {
    if (!a || a->ctx != ctx) return fail(ctx, AIPT_E_INVALID, "aipt_adamw_step: no plan of this context");
    if (!std::isfinite(lr) || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0) || !std::isfinite(eps) || std::isnan(max_norm))
        return fail(ctx, AIPT_E_INVALID, "aipt_adamw_step: lr %g, beta1 %g, beta2 %g, eps %g, max_norm %g", lr, beta1, beta2, eps, max_norm);
    if (!a->grid) return fail(ctx, AIPT_E_INVALID, "aipt_adamw_step: the plan holds no elements");
    aipt::DeviceScope dev(ctx->device);
    AIPT_HIP(ctx, dev.err);
    const bool clip = max_norm > 0;
    aipt::AdamArgs l = a->args;
    const int t = a->grad_type;
    if (clip) {
        aipt::NormKernel k = t == AIPT_TYPE_F32 ? aipt::grad_square<float> : t == AIPT_TYPE_BF16 ? aipt::grad_square<aipt::bf16> : aipt::grad_square<aipt::f16>;
        AIPT_HIP(ctx, aipt::launch(k, a->grid, 256, 0, ctx->stream, aipt::NormArgs{l.tab, l.n, l.blocks, a->partial}));
        l.partial = a->partial; l.npartial = (int)a->grid; l.max_norm = (float)max_norm;
    }
    l.ln1 = std::log(beta1); l.ln2 = std::log(beta2);
    l.lr = (float)lr; l.beta1 = (float)beta1; l.beta2 = (float)beta2; l.eps = (float)eps;
    l.omb1 = (float)(1.0 - beta1); l.omb2 = (float)(1.0 - beta2);
    l.seed = seed;
    aipt::AdamKernel k = t == AIPT_TYPE_F32 ? aipt::adam_of<float>(a->copy_type, a->bits) : t == AIPT_TYPE_BF16 ? aipt::adam_of<aipt::bf16>(a->copy_type, a->bits)
                                                                                               : aipt::adam_of<aipt::f16>(a->copy_type, a->bits);
    AIPT_HIP(ctx, aipt::launch(k, a->grid, 256, 0, ctx->stream, l));
    return AIPT_OK;
}

void aipt_adamw_destroy(aipt_adamw* a) {
    delete a;
}

}  // extern "C"
