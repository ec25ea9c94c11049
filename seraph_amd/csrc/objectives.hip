// objectives.hip - objectives over vocabulary logits beside the cross entropy: log-probabilities of given tokens, the
// clipped policy loss, the paired preference loss and distillation from a teacher's top logits.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "vocab_rows.hpp"

namespace seraph {

constexpr int kBlock = 256;
constexpr int kMaxTopK = 1024;

// What a row's list adds up to: the mass sum q and sum q (log q - (z - at) / T), `at` being the largest listed logit of the
// student (the row's maximum, which the loss needs instead, may not be known yet; differences of logits keep their
// bits also where all of them are masked to the type's lowest value).
struct ListSums { double mass, cross; float at; };

// The gradient of a row, from its statistics: a e + b (second exponential, or e (z - m)), minus c at the target.
struct RowGrad { float a, b, c; int64_t target; };

template <int EXTRA>
__device__ __forceinline__ float grad_at(float z, float m, ExpScale k, const RowGrad& g) {
    const float e = exp_of(z, m, k);
    if (EXTRA == kEntropy) return e == 0.0f ? e * g.a : e * (g.a + g.b * (z - m));
    if (EXTRA == kSecond) return g.a * e + g.b * exp_of(z, m, kUnitScale);
    return g.a * e;
}

// ---------------------------------------------------------------- the objectives
// An objective is a struct of its arguments.  dead(): the outputs of a row that is not supervised.  finish(): called by one lane
// with the statistics of a supervised row; it writes the row's outputs and returns its gradient.  A row's few scalars
// are formed in 64 bits: (z - m) - log(sum) keeps no more than 24 bits of a difference that a ratio of
// log-probabilities needs to more than that, and one lane per row costs nothing beside thousands of logits.
struct LogprobsOp {
    static constexpr bool kGrad = false, kList = false;
    Supervision rows;
    float *logp, *lse, *entropy;
    ExpScale k;
    __device__ __forceinline__ bool live(int64_t r) const { return rows.live(r); }
    __device__ __forceinline__ int64_t target(int64_t r) const { return rows.targets[r]; }
    __device__ __forceinline__ void dead(int64_t r) const {
        logp[r] = 0.0f;
        if (lse) lse[r] = 0.0f;
        if (entropy) entropy[r] = 0.0f;
    }
    template <int EXTRA>
    __device__ __forceinline__ RowGrad finish(int64_t r, RowStats st, float zt, const ListSums&) const {
        const double log_s = log((double)st.s);
        logp[r] = (float)(((double)zt - (double)st.m) - log_s);
        if (lse) lse[r] = (float)((double)st.m + log_s);
        if (EXTRA == kEntropy && entropy) entropy[r] = (float)(log_s - (double)st.x / (double)st.s);
        return RowGrad{0.0f, 0.0f, 0.0f, -1};
    }
};

struct PolicyOp {
    static constexpr bool kGrad = true, kList = false;
    Supervision rows;
    const float *advantages, *old_logp, *ref_logp;
    float *loss_rows, *logp_rows, *kl_rows, *entropy_rows;
    float clip_low, clip_high, kl_coef, entropy_coef, scale;
    ExpScale k;
    __device__ __forceinline__ bool live(int64_t r) const { return rows.live(r); }
    __device__ __forceinline__ int64_t target(int64_t r) const { return rows.targets[r]; }
    __device__ __forceinline__ void dead(int64_t r) const {
        loss_rows[r] = 0.0f;
        if (logp_rows) logp_rows[r] = 0.0f;
        if (kl_rows) kl_rows[r] = 0.0f;
        if (entropy_rows) entropy_rows[r] = 0.0f;
    }
    template <int EXTRA>
    __device__ __forceinline__ RowGrad finish(int64_t r, RowStats st, float zt, const ListSums&) const {
        const double log_s = log((double)st.s), total = (double)st.s;
        const double logp = ((double)zt - (double)st.m) - log_s;
        const double w = rows.weights ? (double)rows.weights[r] : 1.0;
        const double adv = (double)advantages[r];
        const double rho = exp(logp - (double)old_logp[r]);
        const double free = rho * adv;
        const double held = fmin(fmax(rho, 1.0 - (double)clip_low), 1.0 + (double)clip_high) * adv;
        double loss = free > held ? -held : -free;                // NaN takes the second branch of both and stays NaN
        double slope = free > held ? 0.0 : -free;                 // d loss / d logp
        if (ref_logp) {
            const double d = (double)ref_logp[r] - logp;
            const double em1 = expm1(d);
            const double kl = em1 - d;
            if (kl_rows) kl_rows[r] = (float)kl;
            if (kl_coef != 0.0f) {
                loss += (double)kl_coef * kl;
                slope -= (double)kl_coef * em1;
            }
        }
        const double sc = w * (double)scale;
        RowGrad g;
        g.b = 0.0f;
        double a = -slope * sc / total;
        if (EXTRA == kEntropy) {
            const double entropy = log_s - (double)st.x / total;
            if (entropy_rows) entropy_rows[r] = (float)entropy;
            loss -= (double)entropy_coef * entropy;
            a += (double)entropy_coef * sc * (entropy - log_s) / total;     // d(-H)/dz_j = p_j (log p_j + H)
            g.b = (float)((double)entropy_coef * sc / total);
        }
        g.a = (float)a;
        g.c = (float)(-slope * sc);
        g.target = rows.targets[r];
        loss_rows[r] = (float)(w * loss);
        if (logp_rows) logp_rows[r] = (float)logp;
        return g;
    }
};

// One row's list of teacher logits, as the kernels below read it.
struct TeacherList {
    const uint32_t* ids;
    const void* logits;
    const float* lse;              // NULL: the listed logits are the whole distribution
    int type, top_k;
    __device__ __forceinline__ float logit(int64_t i) const {
        if (type == SERAPH_TYPE_F16) return __half2float(reinterpret_cast<const __half*>(logits)[i]);
        if (type == SERAPH_TYPE_BF16) return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(logits)[i] << 16);
        return reinterpret_cast<const float*>(logits)[i];
    }
};

struct DistillOp {
    static constexpr bool kGrad = true, kList = true;
    Supervision rows;              // targets NULL: they do not decide which rows count
    TeacherList list;
    const uint32_t* targets;
    float* loss_rows;
    float soft_coef, hard_coef, scale;
    ExpScale k;
    double inv_temp;
    __device__ __forceinline__ bool live(int64_t r) const { return rows.live(r); }
    __device__ __forceinline__ int64_t target(int64_t r) const {
        if (hard_coef == 0.0f) return -1;
        const int64_t t = targets[r];
        return t < rows.cols ? t : -1;
    }
    __device__ __forceinline__ void dead(int64_t r) const { loss_rows[r] = 0.0f; }
    // what an entry with the part q of the teacher's mass takes off the gradient
    __device__ __forceinline__ float entry_scale(int64_t r) const {
        const double w = rows.weights ? (double)rows.weights[r] : 1.0;
        return (float)(w * (double)scale * (double)soft_coef * inv_temp);
    }
    template <int EXTRA>
    __device__ __forceinline__ RowGrad finish(int64_t r, RowStats st, float zt, const ListSums& list_sums) const {
        const double mass = list_sums.mass;
        const double w = rows.weights ? (double)rows.weights[r] : 1.0;
        const double sc = w * (double)scale;
        const int64_t t = target(r);
        double loss = 0.0, a = 0.0;
        if (soft_coef != 0.0f && mass != 0.0) {
            loss = (double)soft_coef * (list_sums.cross + mass * (((double)st.m - (double)list_sums.at) * inv_temp + log((double)st.s)));
            a = (double)soft_coef * inv_temp * sc * mass / (double)st.s;
        }
        RowGrad g;
        g.b = 0.0f;
        g.c = 0.0f;
        g.target = t;
        if (t >= 0) {
            const double s1 = (double)(EXTRA == kSecond ? st.x : st.s);      // the sum at T = 1
            loss += (double)hard_coef * (log(s1) - ((double)zt - (double)st.m));
            if (EXTRA == kSecond) g.b = (float)((double)hard_coef * sc / s1);
            else a += (double)hard_coef * sc / s1;
            g.c = (float)((double)hard_coef * sc);
        }
        g.a = (float)a;
        loss_rows[r] = (float)(w * loss);
        return g;
    }
};

// ---------------------------------------------------------------- a teacher's list
// Turns a row's list into the mass q of each entry (entries of one id all hold that id's whole mass, added in list order,
// so whichever of them is used last leaves the same value), its logits z, and the row's sums.  Called by a whole
// workgroup; the arrays are its LDS.  The logits are gathered before anything of the row is overwritten.
template <int BLOCK, int K>
struct ListRoom {
    uint32_t id[K];
    float q[K], z[K];
    float red[3][BLOCK / 64];
    double red64[2][BLOCK / 64];
};

template <int BLOCK, int K>
__device__ __forceinline__ ListSums read_list(const TeacherList& l, int64_t r, const float* row, int64_t cols, double inv_temp, ExpScale k, ListRoom<BLOCK, K>& room) {
    const int64_t base = r * l.top_k;
    float m = kLowest, at = kLowest;
    for (int i = threadIdx.x; i < l.top_k; i += BLOCK) {
        const uint32_t id = l.ids[base + i];
        const float u = l.logit(base + i);
        room.id[i] = id;
        room.q[i] = u;
        if ((int64_t)id < cols) {
            const float z = row[id];
            room.z[i] = z;
            m = fmaxf(m, u);
            at = fmaxf(at, z);
        }
    }
    m = block_max<BLOCK>(m, room.red[0]);
    at = block_max<BLOCK>(at, room.red[1]);
    float s = 0.0f;
    for (int i = threadIdx.x; i < l.top_k; i += BLOCK)
        if ((int64_t)room.id[i] < cols) s += exp_of(room.q[i], m, k);
    s = block_sum<BLOCK>(s, room.red[2]);
    // log q_i = (u_i - m) / T + log_norm
    const double log_norm = l.lse ? (double)m * inv_temp - (double)l.lse[r] : -log((double)s);
    const float norm = (float)exp(log_norm);
    ListSums sums{0.0, 0.0, at};
    for (int i = threadIdx.x; i < l.top_k; i += BLOCK) {
        float p = 0.0f;
        if ((int64_t)room.id[i] < cols && s != 0.0f) {            // (no entry at all: no mass, not NaN)
            const float u = room.q[i];
            p = exp_of(u, m, k) * norm;
            if (p != 0.0f)
                sums.cross += (double)p * (((double)u - (double)m) * inv_temp + log_norm - ((double)room.z[i] - (double)at) * inv_temp);
        }
        sums.mass += (double)p;
        room.q[i] = p;
    }
    sums.mass = block_sum<BLOCK>(sums.mass, room.red64[0]);
    sums.cross = block_sum<BLOCK>(sums.cross, room.red64[1]);
    // ids listed twice
    float part[(K + BLOCK - 1) / BLOCK];
#pragma unroll
    for (int j = 0; j < (K + BLOCK - 1) / BLOCK; j++) {
        const int i = threadIdx.x + j * BLOCK;
        part[j] = 0.0f;
        if (i < l.top_k)
            for (int o = 0; o < l.top_k; o++) part[j] += room.id[o] == room.id[i] ? room.q[o] : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < (K + BLOCK - 1) / BLOCK; j++) {
        const int i = threadIdx.x + j * BLOCK;
        if (i < l.top_k) room.q[i] = part[j];
    }
    __syncthreads();
    return sums;
}

// ---------------------------------------------------------------- rows swept from memory
// One workgroup per row: maximum, sums, gradient, each a sweep of its own.
template <class Op, int EXTRA>
__global__ __launch_bounds__(kBlock) void swept_rows_kernel(Op op, const float* logits, float* grad, int64_t cols) {
    __shared__ float red[3][kBlock / 64];
    __shared__ RowGrad bcast;
    __shared__ ListRoom<kBlock, Op::kList ? kMaxTopK : 1> room;
    const int64_t row = blockIdx.x;
    float* out = Op::kGrad ? grad + row * cols : nullptr;
    if (!op.live(row)) {
        if (Op::kGrad) for (int64_t c = threadIdx.x; c < cols; c += kBlock) out[c] = 0.0f;
        if (threadIdx.x == 0) op.dead(row);
        return;
    }
    const float* x = logits + row * cols;
    const ExpScale k = op.k;
    RowStats st;
    float m = kLowest;
    for (int64_t c = threadIdx.x; c < cols; c += kBlock) m = fmaxf(m, x[c]);
    st.m = block_max<kBlock>(m, red[0]);
    float s = 0.0f, ex = 0.0f;
    for (int64_t c = threadIdx.x; c < cols; c += kBlock) {
        const float z = x[c], e = exp_of(z, st.m, k);
        s += e;
        ex += extra_of<EXTRA>(z, st.m, e);
    }
    st.s = block_sum<kBlock>(s, red[1]);
    st.x = EXTRA == kNone ? 0.0f : block_sum<kBlock>(ex, red[2]);
    ListSums sums{0.0, 0.0, 0.0f};
    if constexpr (Op::kList) sums = read_list(op.list, row, x, cols, op.inv_temp, op.k, room);
    if (threadIdx.x == 0) {
        const int64_t t = op.target(row);
        bcast = op.template finish<EXTRA>(row, st, t >= 0 ? x[t] : 0.0f, sums);
    }
    __syncthreads();
    if constexpr (Op::kGrad) {
        const RowGrad g = bcast;
        for (int64_t c = threadIdx.x; c < cols; c += kBlock) {
            const float v = grad_at<EXTRA>(x[c], st.m, k, g);
            out[c] = c == g.target ? v - g.c : v;
        }
        if constexpr (Op::kList) {
            const float es = op.entry_scale(row);
            __syncthreads();                                      // the sweep has written every entry's place
            for (int i = threadIdx.x; i < op.list.top_k; i += kBlock) {
                const uint32_t id = room.id[i];
                if ((int64_t)id < cols) out[id] = grad_at<EXTRA>(room.z[i], st.m, k, g) - es * room.q[i] - ((int64_t)id == g.target ? g.c : 0.0f);
            }
        }
    }
}

template <class Op, int EXTRA>
static int launch_rows(const Op& op, const float* logits, float* grad, int64_t rows, int64_t cols, hipStream_t st) {
    hipLaunchKernelGGL((swept_rows_kernel<Op, EXTRA>), dim3((unsigned)rows), dim3(kBlock), 0, st, op, logits, grad, cols);
    SERAPH_LAUNCH_CHECK();
    return SERAPH_OK;
}

// ---------------------------------------------------------------- preference pairs
struct PreferenceArgs {
    const float* ref_logp;
    float *loss_pairs, *scores, *logp_rows;
    const uint32_t* seq_starts;
    int pairs;
    int64_t rows;
    int kind, average;
    float beta, smoothing, margin;
};

// What the gradient pass needs of a row: its maximum, the factor of exp(z - m), and what the target takes off.
struct RowFactor { float m, a, c; uint32_t target; };
struct RowTotals { float m, s; };

// The statistics of the supervised rows; logp in 64 bits, because a score is a difference of long sums.
struct PairRowsOp {
    static constexpr bool kGrad = false, kList = false;
    Supervision rows;
    RowTotals* totals;
    double* logp;
    RowFactor* factors;
    float* logp_rows;
    ExpScale k;
    __device__ __forceinline__ bool live(int64_t r) const { return rows.live(r); }
    __device__ __forceinline__ int64_t target(int64_t r) const { return rows.targets[r]; }
    __device__ __forceinline__ void dead(int64_t r) const {
        totals[r] = RowTotals{0.0f, 0.0f};
        factors[r] = RowFactor{0.0f, 0.0f, 0.0f, 0xffffffffu};    // target: the row is not supervised
        logp[r] = 0.0;
        if (logp_rows) logp_rows[r] = 0.0f;
    }
    template <int EXTRA>
    __device__ __forceinline__ RowGrad finish(int64_t r, RowStats st, float zt, const ListSums&) const {
        const double v = ((double)zt - (double)st.m) - log((double)st.s);
        totals[r] = RowTotals{st.m, st.s};
        factors[r] = RowFactor{st.m, 0.0f, 0.0f, rows.targets[r]};
        logp[r] = v;
        if (logp_rows) logp_rows[r] = (float)v;
        return RowGrad{0.0f, 0.0f, 0.0f, -1};
    }
};

// One workgroup per pair: the two scores, the loss, and the factor of every row of the pair.
__global__ __launch_bounds__(kBlock) void pair_kernel(PreferenceArgs p, const RowTotals* totals, const double* logp, RowFactor* factors) {
    __shared__ double red[2][kBlock / 64];
    __shared__ double red_n[2][kBlock / 64];
    const int pair = blockIdx.x;
    double score[2], count[2];
    int64_t first[2], last[2];
    for (int side = 0; side < 2; side++) {
        const uint32_t* b = p.seq_starts + 2 * (int64_t)pair + side;
        first[side] = b[0];
        last[side] = (int64_t)b[1] < p.rows ? (int64_t)b[1] : p.rows;
        double sum = 0.0, n = 0.0;
        for (int64_t r = first[side] + threadIdx.x; r < last[side]; r += kBlock)
            if (factors[r].target != 0xffffffffu) {
                sum += p.ref_logp ? logp[r] - (double)p.ref_logp[r] : logp[r];
                n += 1.0;
            }
        score[side] = block_sum<kBlock>(sum, red[side]);
        count[side] = block_sum<kBlock>(n, red_n[side]);
        if (p.average && count[side] > 0.0) score[side] /= count[side];
    }
    const double beta = (double)p.beta, gap = score[0] - score[1], h = beta * gap - (double)p.margin;
    double loss, slope;                                           // slope: d loss / d gap
    if (p.kind == SERAPH_PREFERENCE_SIGMOID) {
        const double eps = (double)p.smoothing, soft = log1p(exp(-fabs(h)));
        loss = (1.0 - eps) * (soft + fmax(-h, 0.0)) + eps * (soft + fmax(h, 0.0));
        if (h != h) loss = h;
        slope = beta * (eps - 1.0 / (1.0 + exp(h)));
    } else if (p.kind == SERAPH_PREFERENCE_HINGE) {
        loss = h >= 1.0 ? 0.0 : 1.0 - h;
        slope = h >= 1.0 ? 0.0 : -beta;
    } else {
        const double d = gap - 0.5 / beta;
        loss = d * d;
        slope = 2.0 * d;
    }
    if (threadIdx.x == 0) {
        p.loss_pairs[pair] = (float)loss;
        if (p.scores) {
            p.scores[2 * (int64_t)pair] = (float)score[0];
            p.scores[2 * (int64_t)pair + 1] = (float)score[1];
        }
    }
    for (int side = 0; side < 2; side++) {
        const double f = (side ? -slope : slope) / (double)p.pairs / (p.average && count[side] > 0.0 ? count[side] : 1.0);
        for (int64_t r = first[side] + threadIdx.x; r < last[side]; r += kBlock)
            if (factors[r].target != 0xffffffffu) {
                factors[r].a = (float)(-f / (double)totals[r].s);
                factors[r].c = (float)-f;
            }
    }
}

__global__ __launch_bounds__(kBlock) void pair_grad_kernel(const float* logits, float* grad, const RowFactor* factors, int64_t cols) {
    const int64_t row = blockIdx.x;
    const RowFactor f = factors[row];
    const float* x = logits + row * cols;
    float* out = grad + row * cols;
    if (f.target == 0xffffffffu) {
        for (int64_t c = threadIdx.x; c < cols; c += kBlock) out[c] = 0.0f;
        return;
    }
    for (int64_t c = threadIdx.x; c < cols; c += kBlock) {
        const float v = f.a * exp_of(x[c], f.m, kUnitScale);
        out[c] = c == (int64_t)f.target ? v - f.c : v;
    }
}

static inline size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace seraph

using namespace seraph;

#define REQUIRE_ROWS(op)                                                                                              \
    SERAPH_REQUIRE(rows > 0 && cols > 0 && rows <= 0x7fffffff && cols <= 0x7fffffff, op ": bad shape %lld x %lld",     \
                   (long long)rows, (long long)cols)
#define REQUIRE_WS(op, need)                                                                                          \
    do {                                                                                                              \
        if ((need) && (!ws || ws_bytes < (need) || !aligned16(ws))) {                                                 \
            set_error(op ": scratch of %zu bytes, 16-byte aligned, needed (given %zu)", (size_t)(need), ws_bytes);     \
            return SERAPH_ERR_WORKSPACE;                                                                              \
        }                                                                                                             \
    } while (0)

extern "C" {

size_t seraph_token_logprobs_ws_bytes(int64_t rows, int64_t cols) {
    (void)rows; (void)cols;
    return 0;
}

int seraph_token_logprobs(const float* logits, const uint32_t* targets, float* logp, float* lse, float* entropy,
                          const uint32_t* seq_starts, int batch, int64_t rows, int64_t cols,
                          void* ws, size_t ws_bytes, seraph_stream_t s) {
    if (rows == 0 || cols == 0) return SERAPH_OK;
    REQUIRE_ROWS("token_logprobs");
    SERAPH_REQUIRE(logits && targets && logp, "token_logprobs: NULL pointer");
    SERAPH_REQUIRE(!seq_starts || batch >= 1, "token_logprobs: packed call needs batch >= 1");
    REQUIRE_WS("token_logprobs", seraph_token_logprobs_ws_bytes(rows, cols));
    LogprobsOp op{{targets, nullptr, seq_starts, batch, cols}, logp, lse, entropy, kUnitScale};
    if (entropy) return launch_rows<LogprobsOp, kEntropy>(op, logits, nullptr, rows, cols, as_stream(s));
    return launch_rows<LogprobsOp, kNone>(op, logits, nullptr, rows, cols, as_stream(s));
}

size_t seraph_policy_grad_ws_bytes(int64_t rows, int64_t cols) {
    (void)rows; (void)cols;
    return 0;
}

int seraph_policy_grad(const float* logits, const uint32_t* actions, const float* advantages, const float* old_logp,
                       const float* ref_logp, const float* weights, float* grad, float* loss_rows,
                       float* logp_rows, float* kl_rows, float* entropy_rows, const seraph_policy_options_t* options,
                       const uint32_t* seq_starts, int batch, int64_t rows, int64_t cols, int64_t valid_rows,
                       void* ws, size_t ws_bytes, seraph_stream_t s) {
    if (rows == 0 || cols == 0) return SERAPH_OK;
    REQUIRE_ROWS("policy_grad");
    SERAPH_REQUIRE(logits && actions && advantages && old_logp && grad && loss_rows && options, "policy_grad: NULL pointer");
    SERAPH_REQUIRE(!seq_starts || batch >= 1, "policy_grad: packed call needs batch >= 1");
    SERAPH_REQUIRE(options->clip_low >= 0.0f && options->clip_high >= 0.0f, "policy_grad: clip bounds %g / %g must not be negative",
                   (double)options->clip_low, (double)options->clip_high);
    SERAPH_REQUIRE(isfinite(options->kl_coef) && isfinite(options->entropy_coef), "policy_grad: coefficients must be finite");
    SERAPH_REQUIRE(ref_logp || (options->kl_coef == 0.0f && !kl_rows), "policy_grad: the KL term needs ref_logp");
    REQUIRE_WS("policy_grad", seraph_policy_grad_ws_bytes(rows, cols));
    const float scale = valid_rows > 0 ? 1.0f / (float)valid_rows : 0.0f;
    PolicyOp op{{actions, weights, seq_starts, batch, cols}, advantages, old_logp, ref_logp, loss_rows, logp_rows, kl_rows, entropy_rows,
                options->clip_low, options->clip_high, options->kl_coef, options->entropy_coef, scale, kUnitScale};
    if (options->entropy_coef != 0.0f || entropy_rows) return launch_rows<PolicyOp, kEntropy>(op, logits, grad, rows, cols, as_stream(s));
    return launch_rows<PolicyOp, kNone>(op, logits, grad, rows, cols, as_stream(s));
}

size_t seraph_preference_grad_ws_bytes(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0) return 0;
    return up16((size_t)rows * sizeof(RowFactor)) + up16((size_t)rows * sizeof(double)) + up16((size_t)rows * sizeof(RowTotals));
}

int seraph_preference_grad(const float* logits, const uint32_t* targets, const float* ref_logp, float* grad,
                           float* loss_pairs, float* scores, float* logp_rows, const seraph_preference_options_t* options,
                           const uint32_t* seq_starts, int pairs, int64_t rows, int64_t cols,
                           void* ws, size_t ws_bytes, seraph_stream_t s) {
    if (rows == 0 || cols == 0) return SERAPH_OK;
    REQUIRE_ROWS("preference_grad");
    SERAPH_REQUIRE(logits && targets && grad && loss_pairs && options && seq_starts, "preference_grad: NULL pointer");
    SERAPH_REQUIRE(pairs > 0 && pairs <= 0x3fffffff, "preference_grad: bad number of pairs %d", pairs);
    SERAPH_REQUIRE(options->kind >= SERAPH_PREFERENCE_SIGMOID && options->kind <= SERAPH_PREFERENCE_SQUARED, "preference_grad: unknown loss %d", options->kind);
    SERAPH_REQUIRE(isfinite(options->beta) && options->beta > 0.0f, "preference_grad: beta %g must be positive", (double)options->beta);
    SERAPH_REQUIRE(options->label_smoothing >= 0.0f && options->label_smoothing <= 1.0f, "preference_grad: label smoothing %g outside [0, 1]", (double)options->label_smoothing);
    SERAPH_REQUIRE(isfinite(options->margin), "preference_grad: margin must be finite");
    REQUIRE_WS("preference_grad", seraph_preference_grad_ws_bytes(rows, cols));
    hipStream_t st = as_stream(s);
    char* p = reinterpret_cast<char*>(ws);
    RowFactor* factors = reinterpret_cast<RowFactor*>(p);
    double* logp = reinterpret_cast<double*>(p += up16((size_t)rows * sizeof(RowFactor)));
    RowTotals* totals = reinterpret_cast<RowTotals*>(p += up16((size_t)rows * sizeof(double)));
    PairRowsOp op{{targets, nullptr, seq_starts, 2 * pairs, cols}, totals, logp, factors, logp_rows, kUnitScale};
    const int rc = launch_rows<PairRowsOp, kNone>(op, logits, nullptr, rows, cols, st);
    if (rc != SERAPH_OK) return rc;
    PreferenceArgs a{ref_logp, loss_pairs, scores, logp_rows, seq_starts, pairs, rows, options->kind, options->average,
                     options->beta, options->label_smoothing, options->margin};
    hipLaunchKernelGGL(pair_kernel, dim3((unsigned)pairs), dim3(kBlock), 0, st, a, totals, logp, factors);
    SERAPH_LAUNCH_CHECK();
    hipLaunchKernelGGL(pair_grad_kernel, dim3((unsigned)rows), dim3(kBlock), 0, st, logits, grad, factors, cols);
    SERAPH_LAUNCH_CHECK();
    return SERAPH_OK;
}

size_t seraph_distill_grad_ws_bytes(int64_t rows, int64_t cols, int64_t top_k) {
    (void)rows; (void)cols; (void)top_k;
    return 0;
}

int seraph_distill_grad(const float* logits, const uint32_t* teacher_ids, const void* teacher_logits, const float* teacher_lse,
                        const uint32_t* targets, const float* weights, float* grad, float* loss_rows,
                        const seraph_distill_options_t* options, const uint32_t* seq_starts, int batch,
                        int64_t rows, int64_t cols, int64_t top_k, int64_t valid_rows,
                        void* ws, size_t ws_bytes, seraph_stream_t s) {
    if (rows == 0 || cols == 0) return SERAPH_OK;
    REQUIRE_ROWS("distill_grad");
    SERAPH_REQUIRE(logits && teacher_ids && teacher_logits && grad && loss_rows && options, "distill_grad: NULL pointer");
    SERAPH_REQUIRE(!seq_starts || batch >= 1, "distill_grad: packed call needs batch >= 1");
    SERAPH_REQUIRE(top_k >= 1 && top_k <= kMaxTopK, "distill_grad: top_k %lld outside 1..%d", (long long)top_k, kMaxTopK);
    SERAPH_REQUIRE(isfinite(options->temperature) && options->temperature >= 1e-3f && options->temperature <= 1e3f,
                   "distill_grad: temperature %g outside [0.001, 1000]", (double)options->temperature);
    SERAPH_REQUIRE(isfinite(options->soft_coef) && isfinite(options->hard_coef), "distill_grad: coefficients must be finite");
    SERAPH_REQUIRE(options->teacher_type >= SERAPH_TYPE_F32 && options->teacher_type <= SERAPH_TYPE_BF16, "distill_grad: unknown teacher type %d", options->teacher_type);
    SERAPH_REQUIRE(targets || options->hard_coef == 0.0f, "distill_grad: the hard part needs targets");
    REQUIRE_WS("distill_grad", seraph_distill_grad_ws_bytes(rows, cols, top_k));
    const float scale = valid_rows > 0 ? 1.0f / (float)valid_rows : 0.0f;
    DistillOp op{{nullptr, weights, seq_starts, batch, cols}, {teacher_ids, teacher_logits, teacher_lse, options->teacher_type, (int)top_k},
                 targets, loss_rows, options->soft_coef, options->hard_coef, scale, ExpScale::of(1.0 / (double)options->temperature), 1.0 / (double)options->temperature};
    // at T = 1 the two parts share their exponentials
    if (options->hard_coef != 0.0f && options->temperature != 1.0f) return launch_rows<DistillOp, kSecond>(op, logits, grad, rows, cols, as_stream(s));
    return launch_rows<DistillOp, kNone>(op, logits, grad, rows, cols, as_stream(s));
}

}  // extern "C"
