// fg_attention_kv8.cu -- tree attention over the 8-bit KV cache: host side,
// the f32 / general kernel and the merge of KV splits.
//
// Per call row and KV head the keys and values are, in order, q_len 8-bit
// slots (visible to every node), tail_len tail slots (visible too) and the
// round's tree nodes at tail slots tail_len + j (node i sees node j iff bit j
// of anc_bits[i] is set).  Nothing outside these slots is read.
#include "fg_common.cuh"

namespace fg {
namespace kv8 {

struct AttnParams {
    const void* q;
    void* out;
    const uint8_t *k8, *v8;
    const float *ks, *vs;
    const void *kt, *vt;  // of the call's layer, like k8, v8, ks, vs
    const int32_t *rows, *q_len, *tail_len;
    const uint32_t* anc;
    int32_t batch, Hkv, D, cap, tcap, N, Hq, G, groups, group_rows, splits, rows_total;
    float scale;
    float *ws_o, *ws_ml;  // [item][split][rows of a group][D], [item][split][{m, l}][rows]
};

// Row b's cache row and lengths; a row or length outside the cache records
// FG_EINVAL and is read as an empty prefix of row 0, which stays in bounds.
struct RowLens {
    int32_t row, q, t;
};
__device__ __forceinline__ RowLens row_lens(const AttnParams& p, int32_t b) {
    RowLens r;
    r.row = cache_row(p.rows, p.batch, b);
    r.q = p.q_len[b];
    r.t = p.tail_len[b];
    const bool ok = r.q >= 0 && r.q <= p.cap && r.q % kBlk == 0 && r.t >= 0 && r.t <= p.tcap - p.N;
    if (!ok && threadIdx.x == 0) atomicCAS(&g_fg_error_word, 0, FG_EINVAL);
    if (!ok || r.row < 0) {
        r.q = r.t = 0;
        r.row = max(r.row, 0);
    }
    return r;
}

__device__ __forceinline__ float e4m3_to_f(uint8_t c) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
    return __half2float(__half(h));
}

}  // namespace kv8
}  // namespace fg

#include "fg_attention_kv8_tc.cu"

namespace fg {
namespace kv8 {

// ---------------------------------------------------------------- general
// 32 query rows x one KV split per CTA; 32 slots at a time are brought to
// shared memory as f32, thread (r, c) of 32 x 4 keeps row r's dims 16 i + 4 c.
constexpr int kGRows = 32;
constexpr int kGLd = kMaxD + 4;

template <typename T>
__global__ void __launch_bounds__(128) attn_general_kernel(const AttnParams p) {
    extern __shared__ float gsm[];
    float* qs = gsm;                    // [32][kGLd]
    float* ks = qs + kGRows * kGLd;     // [32][kGLd]
    float* vs = ks + kBlk * kGLd;       // [32][kGLd]
    float* ps = vs + kBlk * kGLd;       // [32][33]
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int split = blockIdx.x, kvh = blockIdx.y / p.groups, grp = blockIdx.y % p.groups, b = blockIdx.z;
    const int tid = threadIdx.x, r = tid >> 2, c = tid & 3;
    const int D = p.D, row0 = grp * kGRows, R = min(kGRows, p.rows_total - row0);
    const RowLens len = row_lens(p, b);
    const int64_t head = (int64_t)len.row * p.Hkv + kvh;
    const int nq = len.q / kBlk, nt = (len.t + p.N + kBlk - 1) / kBlk, nblk = nq + nt;
    const int per = (nblk + p.splits - 1) / p.splits;
    const int b0 = min(nblk, split * per), b1 = min(nblk, b0 + per);
    for (int e = tid; e < kGRows * D; e += 128) {
        const int rr = e / D, d = e % D;
        const int node = (row0 + rr) / p.G, g = (row0 + rr) % p.G;
        qs[rr * kGLd + d] =
            rr < R ? load_elem(p.q, sizeof(T) == 4 ? FG_DTYPE_F32 : FG_DTYPE_BF16,
                               (((int64_t)b * p.N + node) * p.Hq + kvh * p.G + g) * D + d) : 0.0f;
    }
    const int node = (row0 + min(r, R - 1)) / p.G;
    float m = -INFINITY, l = 0.0f;
    float4 acc[kMaxD / 16];
#pragma unroll
    for (int i = 0; i < kMaxD / 16; ++i) acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int blk = b0; blk < b1; ++blk) {
        __syncthreads();
        const bool is8 = blk < nq;
        const int s0 = is8 ? blk * kBlk : (blk - nq) * kBlk;  // first slot of the block, in its own part
        const int live = is8 ? kBlk : min(kBlk, len.t + p.N - s0);
        if (is8) {
            const float sk = p.ks[head * (p.cap / kBlk) + blk], sv = p.vs[head * (p.cap / kBlk) + blk];
            const int64_t base = (head * p.cap + s0) * D;
            for (int e = tid; e < kBlk * D; e += 128) {
                ks[e / D * kGLd + e % D] = e4m3_to_f(p.k8[base + e]) * sk;
                vs[e / D * kGLd + e % D] = e4m3_to_f(p.v8[base + e]) * sv;
            }
        } else {
            const int64_t base = (head * p.tcap + s0) * D;
            const int32_t dt = sizeof(T) == 4 ? FG_DTYPE_F32 : FG_DTYPE_BF16;
            for (int e = tid; e < kBlk * D; e += 128) {
                const bool in = e / D < live;
                ks[e / D * kGLd + e % D] = in ? load_elem(p.kt, dt, base + e) : 0.0f;
                vs[e / D * kGLd + e % D] = in ? load_elem(p.vt, dt, base + e) : 0.0f;
            }
        }
        __syncthreads();
        float s[kBlk / 4];
#pragma unroll
        for (int j = 0; j < kBlk / 4; ++j) s[j] = 0.0f;
        for (int d = 0; d < D; d += 4) {
            const float4 q4 = *reinterpret_cast<const float4*>(qs + r * kGLd + d);
#pragma unroll
            for (int j = 0; j < kBlk / 4; ++j) {
                const float4 k4 = *reinterpret_cast<const float4*>(ks + (c + 4 * j) * kGLd + d);
                s[j] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[j]))));
            }
        }
        float mx = -INFINITY;
        uint32_t vis = 0;  // slots of the block that row r sees
#pragma unroll
        for (int j = 0; j < kBlk / 4; ++j) {
            const int t = c + 4 * j;
            bool see = t < live;
            if (!is8 && see && s0 + t >= len.t) {
                const int x = s0 + t - len.t;
                see = (p.anc[node * 4 + (x >> 5)] >> (x & 31)) & 1u;
            }
            vis |= (uint32_t)see << t;
            // an infinite score becomes NaN: -inf is what a masked slot has
            s[j] *= p.scale;
            s[j] = see ? fmaf(s[j], 0.0f, s[j]) : -INFINITY;
            mx = fmaxf(mx, s[j]);
        }
        vis |= __shfl_xor_sync(0xffffffffu, vis, 1);
        vis |= __shfl_xor_sync(0xffffffffu, vis, 2);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m, mx);
        const float alpha = m == -INFINITY ? 0.0f : expf(m - mn);
        float part = 0.0f;
#pragma unroll
        for (int j = 0; j < kBlk / 4; ++j) {
            // a masked slot weighs nothing (also where no slot is visible yet: mn = -inf)
            const float e = s[j] == -INFINITY ? 0.0f : expf(s[j] - mn);
            part += e;
            ps[r * 33 + c + 4 * j] = e;
        }
        part += __shfl_xor_sync(0xffffffffu, part, 1);
        part += __shfl_xor_sync(0xffffffffu, part, 2);
        l = l * alpha + part;
        m = mn;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kMaxD / 16; ++i) {
            acc[i].x *= alpha;
            acc[i].y *= alpha;
            acc[i].z *= alpha;
            acc[i].w *= alpha;
        }
        for (int t = 0; t < live; ++t) {
            if (!((vis >> t) & 1u)) continue;  // whatever V holds there
            const float e = ps[r * 33 + t];
#pragma unroll
            for (int i = 0; i < kMaxD / 16; ++i) {
                if (16 * i >= D) break;
                const float4 v4 = *reinterpret_cast<const float4*>(vs + t * kGLd + 16 * i + 4 * c);
                acc[i].x = fmaf(e, v4.x, acc[i].x);
                acc[i].y = fmaf(e, v4.y, acc[i].y);
                acc[i].z = fmaf(e, v4.z, acc[i].z);
                acc[i].w = fmaf(e, v4.w, acc[i].w);
            }
        }
    }
    if (r >= R) return;
    const int item = (b * p.Hkv + kvh) * p.groups + grp;
    if (p.splits > 1) {
        float* ml = p.ws_ml + ((int64_t)item * p.splits + split) * 2 * kGRows;
        if (c == 0) {
            ml[r] = m;
            ml[kGRows + r] = l;
        }
        float* wo = p.ws_o + (((int64_t)item * p.splits + split) * kGRows + r) * D;
#pragma unroll
        for (int i = 0; i < kMaxD / 16; ++i)
            if (16 * i < D) *reinterpret_cast<float4*>(wo + 16 * i + 4 * c) = acc[i];
        return;
    }
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // no visible slot: 0; NaN stays
    const int g = (row0 + r) % p.G;
    T* orow = static_cast<T*>(p.out) + (((int64_t)b * p.N + node) * p.Hq + kvh * p.G + g) * D;
#pragma unroll
    for (int i = 0; i < kMaxD / 16; ++i)
        if (16 * i < D) {
            orow[16 * i + 4 * c] = T(acc[i].x * inv);
            orow[16 * i + 4 * c + 1] = T(acc[i].y * inv);
            orow[16 * i + 4 * c + 2] = T(acc[i].z * inv);
            orow[16 * i + 4 * c + 3] = T(acc[i].w * inv);
        }
}

// out = sum_s e^(m_s - m) O_s / sum_s e^(m_s - m) l_s over the splits of a
// group's rows (natural-log maxima).  One warp per row, fixed order.
template <typename T>
__global__ void __launch_bounds__(128) attn_merge_kernel(const AttnParams p, int32_t group_rows) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const int rr = blockIdx.x * 4 + (threadIdx.x >> 5);  // query row of the KV head
    const int kvh = blockIdx.y, b = blockIdx.z;
    if (rr >= p.rows_total) return;
    const int grp = rr / group_rows, r = rr % group_rows;
    const int64_t item = ((int64_t)b * p.Hkv + kvh) * p.groups + grp;
    const float* ml = p.ws_ml + item * p.splits * 2 * group_rows + r;
    const float* wo = p.ws_o + (item * p.splits * group_rows + r) * p.D;
    float m = -INFINITY;
    for (int s = 0; s < p.splits; ++s) m = fmaxf(m, ml[(int64_t)s * 2 * group_rows]);
    float l = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int d = lane * 4;
    for (int s = 0; s < p.splits; ++s) {
        const float ms = ml[(int64_t)s * 2 * group_rows], ls = ml[(int64_t)s * 2 * group_rows + group_rows];
        // a split without a visible slot holds m = -inf, l = 0, O = 0 (or NaNs that show)
        const float w = ms == -INFINITY ? 1.0f : expf(ms - m);
        l += w * ls;
        if (d < p.D) {
            const float4 o = *reinterpret_cast<const float4*>(wo + (int64_t)s * group_rows * p.D + d);
            acc.x = fmaf(w, o.x, acc.x);
            acc.y = fmaf(w, o.y, acc.y);
            acc.z = fmaf(w, o.z, acc.z);
            acc.w = fmaf(w, o.w, acc.w);
        }
    }
    if (d >= p.D) return;
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
    T* orow = static_cast<T*>(p.out) + (((int64_t)b * p.N + rr / p.G) * p.Hq + kvh * p.G + rr % p.G) * p.D + d;
    orow[0] = T(acc.x * inv);
    orow[1] = T(acc.y * inv);
    orow[2] = T(acc.z * inv);
    orow[3] = T(acc.w * inv);
}

constexpr int kMaxSplits = 64;

struct Plan {
    bool tc;  // tensor-core kernel
    int group_rows, groups, items, splits;
};

// The tensor-core kernel takes head_dim 128 in bf16; f32 and other head_dims
// the general one.
static Plan plan_attn(bool tensor, int32_t B, int32_t N, int32_t Hq, int32_t Hkv, int32_t num_splits, int32_t max_q_len) {
    Plan a;
    const int rows = N * (Hq / Hkv);
    a.tc = tensor;
    if (tensor) {  // groups of 32, 64, 96 or 128 rows, as even as that allows
        a.groups = (rows + 127) / 128;
        a.group_rows = ((rows + a.groups - 1) / a.groups + 31) / 32 * 32;
    } else {
        a.group_rows = kGRows;
        a.groups = (rows + a.group_rows - 1) / a.group_rows;
    }
    a.items = B * Hkv * a.groups;
    if (num_splits > 0) {
        a.splits = num_splits;
    } else if (tensor) {
        // one CTA per SM, at least four tiles each: a split costs its start and the merge (one row of 4096 tokens,
        // 8 heads: 4 / 8 / 16 splits 25.8 / 22.4 / 25.9 us)
        const int64_t tiles = ((int64_t)max_q_len + kBlk + N + kT - 1) / kT;
        int64_t s = 148 / (a.items > 0 ? a.items : 1);
        s = s < tiles / 4 ? s : tiles / 4;
        a.splits = (int)(s < 1 ? 1 : s > kMaxSplits ? kMaxSplits : s);
    } else {
        const int64_t blocks = ((int64_t)max_q_len + kBlk + N + kBlk - 1) / kBlk;
        int64_t s = 4 * 148 / (a.items > 0 ? a.items : 1);
        s = s < blocks / 8 ? s : blocks / 8;
        a.splits = (int)(s < 1 ? 1 : s > kMaxSplits ? kMaxSplits : s);
    }
    return a;
}

// K's or V's codes of one layer as rows of 128 bytes, in boxes of 128 rows.
static bool make_code_map(CUtensorMap* map, const void* codes, uint64_t rows) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[2] = {128, rows < kT ? kT : rows};  // (a smaller cache has no whole tile to load)
    const cuuint64_t strides[1] = {128};
    const cuuint32_t box[2] = {128, (cuuint32_t)kT};
    const cuuint32_t estr[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int NC>
static cudaError_t launch_tc(const AttnParams& p, const Plan& plan, int32_t B, const CUtensorMap& mk,
                             const CUtensorMap& mv, cudaStream_t st) {
    cudaError_t e = cudaFuncSetAttribute(attn_kv8_tc_kernel<NC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         kTcSmem<NC>);
    if (e != cudaSuccess) return e;
    e = launch_pdl(attn_kv8_tc_kernel<NC>, dim3(plan.splits, p.Hkv * plan.groups, B), dim3(kTcThreads), kTcSmem<NC>, st,
                   mk, mv, p);
    if (e != cudaSuccess || plan.splits == 1) return e;
    return launch_pdl(attn_merge_kernel<__nv_bfloat16>, dim3((p.rows_total + 3) / 4, p.Hkv, B), dim3(128), 0, st, p,
                      plan.group_rows);
}

static size_t plan_bytes(const Plan& a, int32_t D) {
    return a.splits <= 1 ? 0 : (size_t)a.items * a.splits * a.group_rows * (size_t)(D + 2) * sizeof(float);
}

template <typename T>
static cudaError_t launch_general(const AttnParams& p, const Plan& plan, int32_t B, cudaStream_t st) {
    const size_t smem = (size_t)(3 * kGRows * kGLd + kGRows * 33) * sizeof(float);
    cudaError_t e = cudaFuncSetAttribute(attn_general_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    if (e != cudaSuccess) return e;
    e = launch_pdl(attn_general_kernel<T>, dim3(plan.splits, p.Hkv * plan.groups, B), dim3(128), smem, st, p);
    if (e != cudaSuccess || plan.splits == 1) return e;
    return launch_pdl(attn_merge_kernel<T>, dim3((p.rows_total + 3) / 4, p.Hkv, B), dim3(128), 0, st, p,
                      plan.group_rows);
}

}  // namespace kv8
}  // namespace fg

using namespace fg;

extern "C" size_t fg_tree_attention_kv8_workspace_size(int32_t B, int32_t n_nodes, int32_t n_q_heads,
                                                       int32_t n_kv_heads, int32_t head_dim, int32_t num_splits,
                                                       int32_t max_q_len) {
    if (B <= 0 || n_nodes <= 0 || n_kv_heads <= 0 || n_q_heads <= 0 || n_q_heads % n_kv_heads || max_q_len < 0 ||
        head_dim <= 0 || num_splits > kv8::kMaxSplits)
        return 0;
    // the size does not depend on the cache's dtype: the larger of the two kernels' needs
    size_t need = kv8::plan_bytes(kv8::plan_attn(false, B, n_nodes, n_q_heads, n_kv_heads, num_splits, max_q_len),
                                  head_dim);
    if (head_dim == 128) {
        const size_t tc = kv8::plan_bytes(
            kv8::plan_attn(true, B, n_nodes, n_q_heads, n_kv_heads, num_splits, max_q_len), head_dim);
        need = tc > need ? tc : need;
    }
    return need;
}

extern "C" fg_status fg_tree_attention_kv8(const void* q, const fg_kv8_cache* cache, int32_t layer,
                                           const int32_t* q_len, const int32_t* tail_len, const uint32_t* anc_bits,
                                           int32_t B, int32_t n_nodes, int32_t n_q_heads, float scale, void* out,
                                           void* workspace, size_t workspace_bytes, int32_t num_splits,
                                           int32_t max_q_len, void* stream) {
    const fg_status s = kv8::check_cache(cache, B);
    if (s != FG_OK) return s;
    if (B == 0) return FG_OK;
    if (!q || !q_len || !tail_len || !anc_bits || !out || layer < 0 || layer >= cache->n_layers || n_nodes <= 0 ||
        n_q_heads <= 0 || n_q_heads % cache->n_kv_heads || max_q_len < 0 || !(scale > 0.0f) || !(scale < INFINITY))
        return FG_EINVAL;
    if (n_nodes > FG_MAX_TREE_NODES || n_nodes > cache->tail_capacity) return FG_ECAPACITY;
    if (num_splits > kv8::kMaxSplits) return FG_EINVAL;
    if (((uintptr_t)q | (uintptr_t)out) % 16) return FG_EINVAL;
    const bool f32 = cache->dtype == FG_DTYPE_F32;
    kv8::AttnParams p = {};
    p.q = q;
    p.out = out;
    const int64_t heads = (int64_t)layer * cache->batch * cache->n_kv_heads;
    const int64_t tail_bytes = heads * cache->tail_capacity * cache->head_dim * (f32 ? 4 : 2);
    p.k8 = (const uint8_t*)cache->k8 + heads * cache->capacity * cache->head_dim;
    p.v8 = (const uint8_t*)cache->v8 + heads * cache->capacity * cache->head_dim;
    p.ks = cache->k_scale + heads * (cache->capacity / kv8::kBlk);
    p.vs = cache->v_scale + heads * (cache->capacity / kv8::kBlk);
    p.kt = (const uint8_t*)cache->k_tail + tail_bytes;
    p.vt = (const uint8_t*)cache->v_tail + tail_bytes;
    p.rows = cache->rows;
    p.q_len = q_len;
    p.tail_len = tail_len;
    p.anc = anc_bits;
    p.batch = cache->batch;
    p.Hkv = cache->n_kv_heads;
    p.D = cache->head_dim;
    p.cap = cache->capacity;
    p.tcap = cache->tail_capacity;
    p.N = n_nodes;
    p.Hq = n_q_heads;
    p.G = n_q_heads / cache->n_kv_heads;
    p.rows_total = n_nodes * p.G;
    p.scale = scale;
    const kv8::Plan plan = kv8::plan_attn(!f32 && p.D == 128, B, n_nodes, n_q_heads, cache->n_kv_heads,
                                          num_splits, max_q_len);
    p.groups = plan.groups;
    p.group_rows = plan.group_rows;
    p.splits = plan.splits;
    if ((int64_t)p.Hkv * p.groups > 65535) return FG_ECAPACITY;
    if (plan.splits > 1) {
        if (!workspace || workspace_bytes < kv8::plan_bytes(plan, p.D) || (uintptr_t)workspace % 16)
            return FG_ECAPACITY;
        p.ws_o = (float*)workspace;
        p.ws_ml = p.ws_o + (size_t)plan.items * plan.splits * plan.group_rows * p.D;
    }
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    if (plan.tc) {
        CUtensorMap mk, mv;
        const uint64_t rows = (uint64_t)p.batch * p.Hkv * p.cap;
        if (!kv8::make_code_map(&mk, p.k8, rows) || !kv8::make_code_map(&mv, p.v8, rows)) return FG_EINVAL;
        e = plan.group_rows == 32   ? kv8::launch_tc<1>(p, plan, B, mk, mv, st)
            : plan.group_rows == 64 ? kv8::launch_tc<2>(p, plan, B, mk, mv, st)
            : plan.group_rows == 96 ? kv8::launch_tc<3>(p, plan, B, mk, mv, st)
                                    : kv8::launch_tc<4>(p, plan, B, mk, mv, st);
    } else {
        e = f32 ? kv8::launch_general<float>(p, plan, B, st) : kv8::launch_general<__nv_bfloat16>(p, plan, B, st);
    }
    if (e != cudaSuccess) {
        set_cuda_error(e);
        return FG_ECUDA;
    }
    return launch_status();
}
