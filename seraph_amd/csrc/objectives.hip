// objectives.hip - objectives over vocabulary logits beside the cross entropy: log-probabilities of given tokens, the
// clipped policy loss, the paired preference loss and distillation from a teacher's top logits.
//
// Which kernel a call takes follows from its columns (and, forward only, its rows):
//   gradient ops      up to 32768 columns: held_rows_kernel (a row in one workgroup's registers)
//                     up to 1245184: shared_rows_kernel (a row in several workgroups' registers)
//                     beyond: swept_rows_kernel (three sweeps over memory)
//   forward only      up to 32768: held_rows_kernel; beyond: streamed_rows_kernel, a row in one run or in several
//   preference        a forward pass, the pairs, and a streaming gradient pass; few rows: the last two in one
#include <atomic>

#include <hip/hip_fp16.h>

#include "vocab_rows.hpp"

namespace seraph {

constexpr int kBlock = 256;
constexpr int kMaxTopK = 1024;
// A launch holds less than 2^32 lanes, of which a row takes 256; those that take 512 (more than 12288 columns) would need more
// than the card's memory before their rows were too many.
constexpr int64_t kMaxRows = 0xffffff;

// What a row's list adds up to: the mass sum q and sum q (log q - (z - at) / T), `at` being the largest listed logit of the
// student (the row's maximum, which the loss needs instead, may not be known yet; differences of logits keep their
// bits also where all of them are masked to the type's lowest value).
struct ListSums { double mass, cross; float at; };

// The gradient of a row, from its statistics: a e + b (second exponential, or e (z - m)), minus c at the target.
struct RowGrad { float a, b, c; int64_t target; };

template <int EXTRA>
__device__ __forceinline__ float grad_at(float z, float m, ExpScale k, const RowGrad& g) {
    const float e = exp_once(z, m, k);
    if (EXTRA == kEntropy) return e == 0.0f ? e * g.a : e * (g.a + g.b * (z - m));
    if (EXTRA == kSecond) return g.a * e + g.b * exp_once(z, m, kUnitScale);
    if (EXTRA == kSquare) return e * (g.a + g.b * e);
    return g.a * e;
}
// the same from the exponential
template <int EXTRA>
__device__ __forceinline__ float grad_of_exp(float e, float a, float b) { return EXTRA == kSquare ? e * (a + b * e) : a * e; }

// ---------------------------------------------------------------- the objectives
// An objective is a struct of its arguments.  dead(): the outputs of a row that is not supervised.  finish(): called by one lane
// with the statistics of a supervised row; it writes the row's outputs (where several workgroups call it, one of them) and
// returns the row's gradient.  A row's log-probability is formed in 64 bits: in FP32 (z - m) - log(sum) keeps 24 bits of a
// value near 10, of which a difference of two log-probabilities, or a sum of hundreds, needs more.
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
    __device__ __forceinline__ RowGrad finish(int64_t r, RowStats st, float zt, const ListSums&, bool writes = true) const {
        const double log_s = log_of_sum(st.s);
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
    __device__ __forceinline__ RowGrad finish(int64_t r, RowStats st, float zt, const ListSums&, bool writes = true) const {
        const double log_s = log_of(st.s);
        const double logp = ((double)zt - (double)st.m) - log_s;
        const float w = rows.weights ? rows.weights[r] : 1.0f, adv = advantages[r];
        const float rho = exp_of((float)(logp - (double)old_logp[r]), 0.0f, kUnitScale);
        // an advantage of 0 stays 0 where the ratio is beyond the type's range (of 64 bits it would not be)
        const bool none = adv == 0.0f && rho == INFINITY;
        const float free = none ? 0.0f : rho * adv;
        const float held = none ? 0.0f : fminf(fmaxf(rho, 1.0f - clip_low), 1.0f + clip_high) * adv;
        float loss = free > held ? -held : -free;                 // NaN takes the second branch of both and stays NaN
        float slope = free > held ? 0.0f : -free;                 // d loss / d logp
        if (ref_logp) {
            const ExpLess kl = exp_less((double)ref_logp[r] - logp);
            if (kl_rows && writes) kl_rows[r] = kl.excess;
            if (kl_coef != 0.0f) {
                loss = fmaf(kl_coef, kl.excess, loss);
                slope = fmaf(-kl_coef, kl.rise, slope);
            }
        }
        const float sc = w * scale, inv_total = 1.0f / st.s;
        RowGrad g{-slope * sc * inv_total, 0.0f, -slope * sc, rows.targets[r]};
        if (EXTRA == kEntropy) {
            const float below = st.x * inv_total;                 // the mean of z - m
            const float entropy = (float)(log_s - (double)below);
            if (entropy_rows && writes) entropy_rows[r] = entropy;
            loss = fmaf(-entropy_coef, entropy, loss);
            g.b = entropy_coef * sc * inv_total;                  // d(-H)/dz_j = p_j (log p_j + H) = p_j ((z_j - m) - below)
            g.a -= g.b * below;
        }
        if (writes) {
            loss_rows[r] = w * loss;
            if (logp_rows) logp_rows[r] = (float)logp;
        }
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
        return (rows.weights ? rows.weights[r] : 1.0f) * scale * soft_coef * (float)inv_temp;
    }
    template <int EXTRA>
    __device__ __forceinline__ RowGrad finish(int64_t r, RowStats st, float zt, const ListSums& list_sums, bool writes = true) const {
        const float w = rows.weights ? rows.weights[r] : 1.0f, sc = w * scale, mass = (float)list_sums.mass;
        RowGrad g{0.0f, 0.0f, 0.0f, target(r)};
        double loss = 0.0;
        if (soft_coef != 0.0f && mass != 0.0f) {
            loss = (double)soft_coef * (list_sums.cross + list_sums.mass * (((double)st.m - (double)list_sums.at) * inv_temp + log_of(st.s)));
            g.a = soft_coef * (float)inv_temp * sc * mass / st.s;
        }
        if (g.target >= 0) {
            const float s1 = EXTRA == kNone ? st.s : st.x;      // the sum at T = 1
            loss += (double)hard_coef * (log_of(s1) - ((double)zt - (double)st.m));
            g.c = hard_coef * sc;
            if (EXTRA == kNone) g.a += g.c / s1;
            else g.b = g.c / s1;
        }
        if (writes) loss_rows[r] = (float)((double)w * loss);
        return g;
    }
};

// ---------------------------------------------------------------- a teacher's list
// A row's list becomes the mass q of each entry, its logits z, gathered before anything of the row is overwritten, and the
// row's sums.  The entries are chained in buckets, so an id listed twice meets itself in its chain.  That is rare, and
// only then are all pairs compared, to add up an id's mass in list order.
//
// Where a workgroup holds a whole row (HELD) all of its waves share the list's work, between the barriers that the row needs
// anyway, and a bucket is a vector of the row: the lane that is about to store a vector finds the entries in it by
// one look.  Of an id listed twice the first entry then takes the whole mass and the others none, so that the order of
// a chain, which is the order of atomics, changes nothing.  Elsewhere one wave does the work, a bucket is a hash of the id,
// and every entry of an id holds the whole mass, so whichever is used last leaves the same value.
//
// The list's LDS is sized by the call: with room for the longest list always, short ones would cost the wave of
// prepare_rows_kernel most of its occupancy.
struct ListRoom {
    float *q, *z;
    uint32_t *id, *next, *first;                                  // next, first: an entry's number plus 1, or 0
    int buckets;
};
static __host__ __device__ inline int hash_buckets(int top_k) {
    int n = 64;
    while (n < top_k) n *= 2;
    return n;
}
static size_t list_bytes(int top_k, int buckets) { return (size_t)(4 * top_k + buckets) * 4; }
__device__ __forceinline__ ListRoom list_room(void* lds, int top_k, int buckets) {
    float* f = reinterpret_cast<float*>(lds);
    uint32_t* u = reinterpret_cast<uint32_t*>(f + 2 * top_k);
    return ListRoom{f, f + top_k, u, u + top_k, u + 2 * top_k, buckets};
}
constexpr uint32_t kNoId = 0xffffffffu;

// 0: the single values ahead of the vectors, 1 + i: vector i, 1 + n4: those behind
__device__ __forceinline__ int held_bucket(const RowShape& sh, uint32_t id) {
    const int i4 = ((int)id - sh.head) >> 2;
    return (int)id < sh.head ? 0 : i4 < sh.n4 ? 1 + i4 : 1 + sh.n4;
}
__device__ __forceinline__ int hashed_bucket(const ListRoom& room, uint32_t id) { return (int)((id * 2654435761u) >> 8 & (uint32_t)(room.buckets - 1)); }

__device__ __forceinline__ bool meets_itself(const ListRoom& room, int i, int bucket) {
    bool twice = false;
    for (uint32_t o = room.first[bucket]; o; o = room.next[o - 1]) twice |= o != (uint32_t)i + 1u && room.id[o - 1] == room.id[i];
    return twice;
}
// the mass of entry i's id; `first`: none where an earlier entry has it
__device__ __forceinline__ float mass_of_id(const ListRoom& room, int n, int i, bool first) {
    float sum = 0.0f;
    for (int o = 0; o < n; o++)
        if (room.id[o] == room.id[i]) {
            if (first && o < i) return 0.0f;
            sum += room.q[o];
        }
    return sum;
}

// log q_i = (u_i - m) / T + log; q sums up to s exp(log), which is 1 where the list is the whole distribution
struct ListNorm { double log; float factor; double mass; };
__device__ __forceinline__ ListNorm list_norm(const TeacherList& l, int64_t r, float m, float s, double inv_temp) {
    ListNorm o;
    o.log = l.lse ? (double)m * inv_temp - (double)l.lse[r] : -log_of(s);
    o.factor = l.lse ? exp_of((float)o.log, 0.0f, kUnitScale) : 1.0f / s;
    o.mass = s == 0.0f ? 0.0 : l.lse ? (double)s * (double)o.factor : s == s ? 1.0 : (double)s;      // (no entry at all: no mass, not NaN)
    return o;
}
// what an entry of mass p adds to the sum q (log q - (z - at) / T)
__device__ __forceinline__ double cross_part(float p, float u, float m, float z, float at, double inv_temp, double log_norm) {
    return p == 0.0f ? 0.0 : (double)p * (((double)u - (double)m) * inv_temp + log_norm - ((double)z - (double)at) * inv_temp);
}

__device__ __forceinline__ void wave_sync() {                     // the wave's own LDS writes are complete and in order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// One wave's form.
__device__ __forceinline__ ListSums read_list(const TeacherList& l, int64_t r, const float* row, int64_t cols, double inv_temp, ExpScale k, const ListRoom& room) {
    const int lane = (int)threadIdx.x & 63, n = l.top_k;
    const int64_t base = r * n;
    float m = kLowest, at = kLowest;
    for (int i = lane; i < room.buckets; i += 64) room.first[i] = 0u;
    wave_sync();
    constexpr int kAhead = 4;                                     // entries in flight per lane: a list of 256 waits for memory twice
    for (int i0 = lane; i0 < n; i0 += 64 * kAhead) {
        uint32_t id[kAhead];
        float u[kAhead], z[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const int i = i0 + j * 64;
            id[j] = i < n ? l.ids[base + i] : kNoId;
            u[j] = i < n ? l.logit(base + i) : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            if ((int64_t)id[j] >= cols) id[j] = kNoId;
            z[j] = id[j] != kNoId ? row[id[j]] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const int i = i0 + j * 64;
            if (i >= n) break;
            room.id[i] = id[j];
            room.q[i] = u[j];
            room.z[i] = z[j];
            if (id[j] != kNoId) {
                room.next[i] = atomicExch(&room.first[hashed_bucket(room, id[j])], (uint32_t)i + 1u);
                m = fmaxf(m, u[j]);
                at = fmaxf(at, z[j]);
            }
        }
    }
    wave_sync();
    bool twice = false;
    for (int i = lane; i < n; i += 64)
        if (room.id[i] != kNoId) twice |= meets_itself(room, i, hashed_bucket(room, room.id[i]));
    twice = __any(twice);
    m = wave_top(m);
    at = wave_top(at);
    float s = 0.0f;
    for (int i = lane; i < n; i += 64)
        if (room.id[i] != kNoId) s += exp_of(room.q[i], m, k);
    s = wave_total(s);
    const ListNorm norm = list_norm(l, r, m, s, inv_temp);
    double cross = 0.0;
    for (int i = lane; i < n; i += 64) {
        const float u = room.q[i], p = room.id[i] != kNoId && s != 0.0f ? exp_of(u, m, k) * norm.factor : 0.0f;
        cross += cross_part(p, u, m, room.z[i], at, inv_temp, norm.log);
        room.q[i] = p;
    }
    cross = wave_total(cross);
    if (twice) {
        wave_sync();
        float part[kMaxTopK / 64];
#pragma unroll
        for (int j = 0; j < kMaxTopK / 64; j++) part[j] = lane + j * 64 < n ? mass_of_id(room, n, lane + j * 64, false) : 0.0f;
        wave_sync();
#pragma unroll
        for (int j = 0; j < kMaxTopK / 64; j++)
            if (lane + j * 64 < n) room.q[lane + j * 64] = part[j];
    }
    wave_sync();
    return ListSums{norm.mass, cross, at};
}

// ---------------------------------------------------------------- rows held in registers
// One workgroup owns a row of up to 4 kBlock VPT columns (and seven single values) and holds it in its registers: a logit
// crosses memory once in each direction.
// Waves per SIMD asked for: at eight, all of 2048 rows of 8192 columns are on the chip at once (21.4 us; at six 24.7 us); the
// list ops would spill.
constexpr int held_waves(int vpt, bool list) { return list ? 4 : vpt <= 8 ? 8 : vpt <= 12 ? 5 : 4; }
template <class Op, int EXTRA, int BLOCK, int VPT>
__global__ __launch_bounds__(BLOCK, held_waves(VPT, Op::kList)) void held_rows_kernel(Op op, const float* logits, float* grad, int cols) {
    __shared__ float red[3][BLOCK / 64];
    __shared__ RowGrad bcast;
    __shared__ float list_red[3][BLOCK / 64];
    __shared__ double list_cross[BLOCK / 64];
    __shared__ int listed_twice;
    extern __shared__ char list_lds[];
    const int64_t row = blockIdx.x;
    const float* x = logits + row * cols;
    float* out = Op::kGrad ? grad + row * cols : nullptr;
    const RowShape sh(x, cols);
    const int single = (int)sh.single((int)threadIdx.x);
    const SlotBuffer xs(x + sh.head, sh.n4);
    if (!op.live(row)) {
        if constexpr (Op::kGrad) {
            const SlotBuffer gs(out + sh.head, sh.n4);
#pragma unroll
            for (int k = 0; k < VPT; k++) gs.store<kNontemporal>(f4{0, 0, 0, 0}, (k * BLOCK + (int)threadIdx.x) * 16);
            if (single >= 0) out[single] = 0.0f;
        }
        if (threadIdx.x == 0) op.dead(row);
        return;
    }
    // a list's ids and logits are asked for ahead of the row, and the row's logits at its ids behind it: memory answers in order
    constexpr int kEntries = kMaxTopK / BLOCK;
    uint32_t id[Op::kList ? kEntries : 1];
    float u[Op::kList ? kEntries : 1];
    ListRoom room{};
    if constexpr (Op::kList) {
        room = list_room(list_lds, op.list.top_k, sh.n4 + 2);
#pragma unroll
        for (int j = 0; j < kEntries; j++) {
            const int i = j * BLOCK + (int)threadIdx.x;
            id[j] = i < op.list.top_k ? op.list.ids[row * op.list.top_k + i] : kNoId;
            u[j] = i < op.list.top_k ? op.list.logit(row * op.list.top_k + i) : 0.0f;
        }
        for (int i = threadIdx.x; i < room.buckets; i += BLOCK) room.first[i] = 0u;
        if (threadIdx.x == 0) listed_twice = 0;
    }
    f4 v[VPT];
#pragma unroll
    for (int k = 0; k < VPT; k++) v[k] = xs.load<kNontemporal>((k * BLOCK + (int)threadIdx.x) * 16);
    float one = single >= 0 ? x[single] : -INFINITY;
    float zt = 0.0f;
    if (threadIdx.x == 0) {
        const int64_t t = op.target(row);
        if (t >= 0) zt = x[t];
    }
    float lm = kLowest, at = kLowest;
    if constexpr (Op::kList) {
#pragma unroll
        for (int j = 0; j < kEntries; j++) {
            const int i = j * BLOCK + (int)threadIdx.x;
            if (i >= op.list.top_k) break;
            if ((int64_t)id[j] >= cols) id[j] = kNoId;
            room.id[i] = id[j];
            room.q[i] = u[j];
            if (id[j] != kNoId) {
                const float z = x[id[j]];
                room.z[i] = z;
                lm = fmaxf(lm, u[j]);
                at = fmaxf(at, z);
            }
        }
        lm = wave_top(lm);
        at = wave_top(at);
        if ((threadIdx.x & 63) == 0) {
            list_red[0][threadIdx.x >> 6] = lm;
            list_red[1][threadIdx.x >> 6] = at;
        }
    }
    const ExpScale ks = op.k;
    float m = fmaxf(kLowest, one);
#pragma unroll
    for (int k = 0; k < VPT; k++) {
        if (k * BLOCK + (int)threadIdx.x >= sh.n4) v[k] = f4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        m = fmaxf(m, fmaxf(fmaxf(v[k].x, v[k].y), fmaxf(v[k].z, v[k].w)));
    }
    m = block_max<BLOCK>(m, red[0]);
    if constexpr (Op::kList) {                                    // the buckets are clear, the list's maxima complete
#pragma unroll
        for (int w = 0; w < BLOCK / 64; w++) { lm = fmaxf(lm, list_red[0][w]); at = fmaxf(at, list_red[1][w]); }
        float part = 0.0f;
        for (int i = threadIdx.x; i < op.list.top_k; i += BLOCK)
            if (room.id[i] != kNoId) {
                room.next[i] = atomicExch(&room.first[held_bucket(sh, room.id[i])], (uint32_t)i + 1u);
                part += exp_of(room.q[i], lm, ks);
            }
        part = wave_total(part);
        if ((threadIdx.x & 63) == 0) list_red[2][threadIdx.x >> 6] = part;
    }
    float e1 = exp_of(one, m, ks), s = e1, ex = EXTRA != kNone ? extra_of<EXTRA>(one, m, e1) : 0.0f;
#pragma unroll
    for (int k = 0; k < VPT; k++) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const float e = exp_of(v[k][c], m, ks);
            s += e;
            if (EXTRA != kNone) ex += extra_of<EXTRA>(v[k][c], m, e);
            if (Op::kGrad && holds_exp(EXTRA)) v[k][c] = e;
        }
        if (!Op::kList) asm volatile("" : "+v"(v[k]));            // four values stay the four registers that a store takes
    }
    if (EXTRA != kNone) block_sum2<BLOCK>(s, ex, red[1]);
    else s = block_sum<BLOCK>(s, red[1]);
    const RowStats stats{m, s, ex};
    ListSums sums{0.0, 0.0, at};
    if constexpr (Op::kList) {                                    // the chains and the list's sum are complete
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < BLOCK / 64; w++) total += list_red[2][w];
        const ListNorm norm = list_norm(op.list, row, lm, total, op.inv_temp);
        sums.mass = norm.mass;
        double cross = 0.0;
        bool twice = false;
        for (int i = threadIdx.x; i < op.list.top_k; i += BLOCK) {
            float p = 0.0f;
            if (room.id[i] != kNoId) {
                p = total != 0.0f ? exp_of(room.q[i], lm, ks) * norm.factor : 0.0f;
                cross += cross_part(p, room.q[i], lm, room.z[i], at, op.inv_temp, norm.log);
                twice |= meets_itself(room, i, held_bucket(sh, room.id[i]));
            }
            room.q[i] = p;
        }
        cross = wave_total(cross);
        if ((threadIdx.x & 63) == 0) list_cross[threadIdx.x >> 6] = cross;
        if (__any(twice) && (threadIdx.x & 63) == 0) listed_twice = 1;
    }
    if (threadIdx.x == 0) bcast = op.template finish<EXTRA>(row, stats, zt, sums, !Op::kList);
    if constexpr (Op::kList) {
        __syncthreads();
        if (threadIdx.x == 0) {                                   // the loss is the one thing that needs the last sum
            for (int w = 0; w < BLOCK / 64; w++) sums.cross += list_cross[w];
            op.template finish<EXTRA>(row, stats, zt, sums, true);
        }
        if (listed_twice) {                                       // (the same for the whole workgroup)
            float part[kEntries];
#pragma unroll
            for (int j = 0; j < kEntries; j++) {
                const int i = j * BLOCK + (int)threadIdx.x;
                part[j] = i < op.list.top_k ? mass_of_id(room, op.list.top_k, i, true) : 0.0f;
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < kEntries; j++)
                if (j * BLOCK + (int)threadIdx.x < op.list.top_k) room.q[j * BLOCK + (int)threadIdx.x] = part[j];
        }
    }
    if constexpr (Op::kGrad) {
        if (!Op::kList || listed_twice) __syncthreads();
        const RowGrad g = bcast;
        const SlotBuffer gs(out + sh.head, sh.n4);
        float es = 0.0f;
        if constexpr (Op::kList) es = op.entry_scale(row);
        const int tv = (int)g.target - sh.head, t4 = g.target >= sh.head ? tv >> 2 : -1;      // the target's place among the vectors
        const f4 off_target = {(tv & 3) == 0 ? g.c : 0.0f, (tv & 3) == 1 ? g.c : 0.0f, (tv & 3) == 2 ? g.c : 0.0f, (tv & 3) == 3 ? g.c : 0.0f};
        if (!holds_exp(EXTRA)) asm volatile("" : "+v"(m));        // the sums' exponentials are not to be kept for here
#pragma unroll
        for (int k = 0; k < VPT; k++) {
            const int i4 = k * BLOCK + (int)threadIdx.x;
            f4 r;
#pragma unroll
            for (int c = 0; c < 4; c++) r[c] = holds_exp(EXTRA) ? grad_of_exp<EXTRA>(v[k][c], g.a, g.b) : grad_at<EXTRA>(v[k][c], m, ks, g);
            if (t4 == i4) r -= off_target;
            if constexpr (Op::kList) {
                for (uint32_t o = i4 < sh.n4 ? room.first[1 + i4] : 0u; o; o = room.next[o - 1]) {
                    const int c = ((int)room.id[o - 1] - sh.head) & 3;
                    const float q = es * room.q[o - 1];
                    r -= f4{c == 0 ? q : 0.0f, c == 1 ? q : 0.0f, c == 2 ? q : 0.0f, c == 3 ? q : 0.0f};
                }
            }
            gs.store<kNontemporal>(r, i4 * 16);
        }
        if (single >= 0) {
            float r = grad_at<EXTRA>(one, m, ks, g);
            if (single == g.target) r -= g.c;
            if constexpr (Op::kList)
                for (uint32_t o = room.first[single < sh.head ? 0 : 1 + sh.n4]; o; o = room.next[o - 1])
                    if (room.id[o - 1] == (uint32_t)single) r -= es * room.q[o - 1];
            out[single] = r;
        }
    }
}

// ---------------------------------------------------------------- long rows shared out between workgroups
// A row that one workgroup's registers cannot hold is cut into chunks of 4 KB (one vector per lane of a workgroup); chunk c
// belongs to part c % P, and P workgroups hold one part each, kPartVpt vectors per lane, so that a logit still crosses
// memory once in each direction.  Each publishes its part's maximum and sums in a record in device memory and combines
// the row's P records by itself in one fixed order, so all of them arrive at the same bits.
//
// The grid is persistent (a multiple of P, at most kPartsPerCu workgroups on a CU); workgroup g takes units g, g + G, ...,
// unit u being part u % P of row u / P, and loads its next unit's slots as it stores this one's.  A small kernel ahead of this
// one clears the records (nothing is carried over from another call or from an earlier replay of a captured one) and
// gathers what belongs to a row as a whole: its target's logit and its list.
//
// The wait for a partner's record is bounded.  Past the limit a workgroup forms the missing part's statistics from the
// logits, with the owner's slots per lane and order of additions, hence to the owner's bits; and if the record has
// appeared meanwhile it takes that, because in place the owner may by then be overwriting those logits (it
// publishes before it stores).  So no workgroup ever depends on another one being scheduled.
constexpr int kPartVpt = 19;                 // 76 of the 128 registers that a lane has with four workgroups on a CU
constexpr int kPartsPerCu = 4;
constexpr int kMaxParts = 64;                // one lane of the first wave per partner

// Each word carries its own validity in its upper half, so no order between the words is needed, hence no fence (which
// at this scope would write back and invalidate whole caches): relaxed device-scope atomics go past the XCDs' L2s.
struct PartRecord { unsigned long long max_word, sum_word, extra_word, unused; };
constexpr unsigned long long kPublished = 1ull << 32;

struct RowPrep { ListSums sums; float zt; int live; };

__device__ __forceinline__ void put_word(unsigned long long* w, float v) {
    __hip_atomic_store(w, kPublished | __float_as_uint(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <int EXTRA>
__device__ __forceinline__ bool get_record(PartRecord* rec, RowStats& st) {
    const unsigned long long a = __hip_atomic_load(&rec->max_word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const unsigned long long b = __hip_atomic_load(&rec->sum_word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const unsigned long long c = EXTRA == kNone ? kPublished : __hip_atomic_load(&rec->extra_word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const bool ok = (a & b & c & kPublished) != 0;
    st.m = ok ? __uint_as_float((unsigned)a) : st.m;
    st.s = ok ? __uint_as_float((unsigned)b) : st.s;
    st.x = ok ? __uint_as_float((unsigned)c) : st.x;
    return ok;
}

// a part's sums against the row's maximum m
template <int EXTRA>
__device__ __forceinline__ RowStats against(RowStats st, float m, ExpScale k) {
    const float r = exp_of(st.m, m, k);
    RowStats o{m, st.s == 0.0f ? 0.0f : st.s * r, 0.0f};
    if (EXTRA == kEntropy) o.x = st.s == 0.0f || r == 0.0f ? 0.0f : (st.x + (st.m - m) * st.s) * r;
    if (EXTRA == kSecond || EXTRA == kSquare) o.x = st.x == 0.0f ? 0.0f : st.x * exp_of(st.m, m, kUnitScale);
    return o;
}

// Clears the rows' records and gathers what belongs to a row as a whole.  A wave takes kPrepRows rows, a lane each, or, of an
// op with lists, one row.
constexpr int kPrepRows = 16;
template <class Op>
__global__ __launch_bounds__(64) void prepare_rows_kernel(Op op, const float* logits, int64_t rows, int64_t cols, int P, RowPrep* prep,
                                                          PartRecord* records, float* list_q, float* list_z) {
    constexpr int kTake = Op::kList ? 1 : kPrepRows;
    const int64_t first = (int64_t)blockIdx.x * kTake;
    const int here = rows - first < kTake ? (int)(rows - first) : kTake;
    unsigned long long* words = reinterpret_cast<unsigned long long*>(records + first * P);
    for (int i = threadIdx.x; i < here * P * 4; i += 64) __hip_atomic_store(words + i, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if constexpr (Op::kList) {
        extern __shared__ char list_lds[];
        const ListRoom room = list_room(list_lds, op.list.top_k, hash_buckets(op.list.top_k));
        ListSums sums{0.0, 0.0, 0.0f};
        const int64_t row = first;
        const float* x = logits + row * cols;
        const bool live = op.live(row);
        if (live) {
            sums = read_list(op.list, row, x, cols, op.inv_temp, op.k, room);
            for (int i = threadIdx.x; i < op.list.top_k; i += 64) {
                list_q[row * op.list.top_k + i] = room.q[i];
                list_z[row * op.list.top_k + i] = room.z[i];
            }
        }
        if (threadIdx.x == 0) {
            const int64_t t = live ? op.target(row) : -1;
            prep[row] = RowPrep{sums, t >= 0 ? x[t] : 0.0f, live ? 1 : 0};
        }
    } else if ((int)threadIdx.x < here) {
        const int64_t row = first + threadIdx.x;
        const bool live = op.live(row);
        const int64_t t = live ? op.target(row) : -1;
        prep[row] = RowPrep{{0.0, 0.0, 0.0f}, t >= 0 ? logits[row * cols + t] : 0.0f, live ? 1 : 0};
    }
}

template <class Op, int EXTRA>
__global__ __launch_bounds__(kBlock, kPartsPerCu) void shared_rows_kernel(Op op, const float* logits, float* grad, int rows, int64_t cols, int P,
                                                                          const RowPrep* prep, PartRecord* records, const float* list_q,
                                                                          const float* list_z, int spin_limit, int in_place) {
    __shared__ float red[3][kBlock / 64];
    __shared__ RowStats parts[kMaxParts];
    __shared__ unsigned long long missing;
    __shared__ struct { RowGrad g; RowStats st; } bcast;
    const int part = (int)(blockIdx.x % (unsigned)P), stride = (int)(gridDim.x / (unsigned)P);
    const ExpScale ks = op.k;
    const f4 pad = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};

    // The entries of a list that lie in this part replace what the dense stores left at their places.  Called behind a
    // barrier that every wave of the workgroup reaches with its stores complete.
    auto write_entries = [&](int64_t row, const RowGrad& g, float m) {
        if constexpr (Op::kList) {
            float* out = grad + row * cols;
            const int head = RowShape(logits + row * cols, cols).head, n4 = RowShape(logits + row * cols, cols).n4;
            const float es = op.entry_scale(row);
            const int64_t base = row * op.list.top_k;
            for (int i = threadIdx.x; i < op.list.top_k; i += kBlock) {
                const uint32_t id = op.list.ids[base + i];
                if ((int64_t)id >= cols) continue;
                const int i4 = ((int)id - head) >> 2;
                const int owner = (int)id < head || i4 >= n4 ? 0 : (i4 / kBlock) % P;
                if (owner == part)
                    out[id] = grad_at<EXTRA>(list_z[base + i], m, ks, g) - es * list_q[base + i] - ((int64_t)id == g.target ? g.c : 0.0f);
            }
        }
    };

    // A lane's slots lie step_bytes apart.  The offset runs: kept opaque, so that the compiler does not hold one register
    // per slot over the whole kernel.
    const int lane_bytes = (part * kBlock + (int)threadIdx.x) * 16, step_bytes = P * kBlock * 16;
#define SERAPH_NEXT_SLOT(off) do { off += step_bytes; asm volatile("" : "+v"(off)); } while (0)
    // the next row from r on that is supervised; the rows passed over get their zeros
    auto next_live = [&](int r) {
        for (; r < rows && !__builtin_amdgcn_readfirstlane(prep[r].live); r += stride) {
            float* out = grad + (int64_t)r * cols;
            const RowShape sh(logits + (int64_t)r * cols, cols);
            const SlotBuffer gs(out + sh.head, sh.n4);
            int off = lane_bytes;
#pragma unroll 1
            for (int k = 0; k < kPartVpt; k++) { gs.store<kNontemporal>(f4{0, 0, 0, 0}, off); off += step_bytes; }
            const int64_t single = part == 0 ? sh.single((int)threadIdx.x) : -1;
            if (single >= 0) out[single] = 0.0f;
            if (part == 0 && threadIdx.x == 0) op.dead(r);
        }
        return r;
    };
    int row = next_live((int)(blockIdx.x / (unsigned)P));
    if (row >= rows) return;
    f4 v[kPartVpt];
    float one;
    {
        const float* x = logits + (int64_t)row * cols;
        const RowShape sh(x, cols);
        const SlotBuffer xs(x + sh.head, sh.n4);
        int off = lane_bytes;
#pragma unroll
        for (int k = 0; k < kPartVpt; k++) { v[k] = xs.load<kNontemporal>(off); SERAPH_NEXT_SLOT(off); }
        const int64_t c = part == 0 ? sh.single((int)threadIdx.x) : -1;
        one = c >= 0 ? x[c] : -INFINITY;
    }
    for (int listed = -1;;) {                                     // listed: a row whose entries are still to be written
        const float* x = logits + (int64_t)row * cols;
        float* out = grad + (int64_t)row * cols;
        const RowShape sh(x, cols);
        float m = fmaxf(kLowest, one);
        {
            const int end = sh.n4 * 16;
            int off = lane_bytes;
#pragma unroll
            for (int k = 0; k < kPartVpt; k++) {
                if (off >= end) v[k] = pad;
                m = fmaxf(m, fmaxf(fmaxf(v[k].x, v[k].y), fmaxf(v[k].z, v[k].w)));
                SERAPH_NEXT_SLOT(off);
            }
        }
        if (Op::kList) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        RowStats mine{block_max<kBlock>(m, red[0]), 0.0f, 0.0f};
        if (Op::kList && listed >= 0) write_entries(listed, bcast.g, bcast.st.m);
        const float e1 = exp_of(one, mine.m, ks);
        float s = e1, ex = EXTRA != kNone ? extra_of<EXTRA>(one, mine.m, e1) : 0.0f;
#pragma unroll
        for (int k = 0; k < kPartVpt; k++) {
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const float e = exp_of(v[k][c], mine.m, ks);
                s += e;
                if (EXTRA != kNone) ex += extra_of<EXTRA>(v[k][c], mine.m, e);
                if (holds_exp(EXTRA)) v[k][c] = e;
            }
            asm volatile("" : "+v"(v[k]));                        // four exponentials stay the four registers that a store takes
        }
        if (EXTRA != kNone) block_sum2<kBlock>(s, ex, red[1]);
        else s = block_sum<kBlock>(s, red[1]);
        mine.s = s;
        mine.x = ex;

        // The first wave, one lane per part, waits for the row's records (once more, over `parts`, where one was missing).
        PartRecord* recs = records + (int64_t)row * P;
        for (bool again = false;; again = true) {
            if (threadIdx.x < 64) {
                const int lane = (int)threadIdx.x;
                RowStats got{kLowest, 0.0f, 0.0f};
                bool ok = lane >= P;
                if (!again) {
                    if (lane == 0) {
                        put_word(&recs[part].max_word, mine.m);
                        put_word(&recs[part].sum_word, mine.s);
                        if (EXTRA != kNone) put_word(&recs[part].extra_word, mine.x);
                        // in place this part's logits are about to be overwritten: the record is out before that
                        if (in_place) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    }
                    if (!ok) ok = get_record<EXTRA>(recs + lane, got);
                    for (int spin = 0; !ok && spin < spin_limit; spin++) {
                        __builtin_amdgcn_s_sleep(4);
                        ok = get_record<EXTRA>(recs + lane, got);
                    }
                } else if (!ok) {
                    got = parts[lane];
                    ok = true;
                }
                const unsigned long long todo = __ballot(!ok);
                if (lane == 0) missing = todo;
                if (todo) {
                    if (lane < P) parts[lane] = got;
                } else {
                    const float rm = wave_top(got.m);
                    const RowStats o = against<EXTRA>(got, rm, ks);
                    const RowStats total{rm, wave_total(o.s), EXTRA != kNone ? wave_total(o.x) : 0.0f};
                    if (lane == 0) {
                        bcast.st = total;
                        bcast.g = op.template finish<EXTRA>(row, total, prep[row].zt, prep[row].sums, part == 0);
                    }
                }
            }
            __syncthreads();
            unsigned long long todo = missing;                    // the same value for the whole workgroup
            if (!todo) break;
            const SlotBuffer xs(x + sh.head, sh.n4);
            while (todo) {
                const int p = __builtin_ctzll(todo);
                todo &= todo - 1;
                const int64_t c1 = p == 0 ? sh.single((int)threadIdx.x) : -1;
                const float o1 = c1 >= 0 ? x[c1] : -INFINITY;
                float pm = fmaxf(kLowest, o1);
                __syncthreads();                                  // red and missing have been read
#pragma unroll 1
                for (int k = 0; k < kPartVpt; k++) {
                    const int i4 = (p + k * P) * kBlock + (int)threadIdx.x;
                    const f4 w = i4 < sh.n4 ? xs.load<0>(i4 * 16) : pad;
                    pm = fmaxf(pm, fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w)));
                }
                RowStats st{block_max<kBlock>(pm, red[0]), 0.0f, 0.0f};
                const float f1 = exp_of(o1, st.m, ks);
                float ps = f1, px = EXTRA != kNone ? extra_of<EXTRA>(o1, st.m, f1) : 0.0f;
#pragma unroll 1
                for (int k = 0; k < kPartVpt; k++) {
                    const int i4 = (p + k * P) * kBlock + (int)threadIdx.x;
                    const f4 w = i4 < sh.n4 ? xs.load<0>(i4 * 16) : pad;
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const float e = exp_of(w[c], st.m, ks);
                        ps += e;
                        if (EXTRA != kNone) px += extra_of<EXTRA>(w[c], st.m, e);
                    }
                }
                if (EXTRA != kNone) block_sum2<kBlock>(ps, px, red[1]);
                else ps = block_sum<kBlock>(ps, red[1]);
                st.s = ps;
                st.x = px;
                if (threadIdx.x == 0) {                           // (behind the reductions' barriers every lane's loads have returned)
                    get_record<EXTRA>(recs + p, st);
                    parts[p] = st;
                }
            }
            __syncthreads();
        }
        const RowGrad g = bcast.g;
        float rm = bcast.st.m;
        if (!holds_exp(EXTRA)) asm volatile("" : "+v"(rm));       // the sums' exponentials are not to be kept for here
        const float up = holds_exp(EXTRA) ? exp_of(mine.m, rm, ks) : 0.0f;      // this part's exponentials against the row's maximum
        const float ga = g.a * up, gb = g.b * up * up;
        const int tv = (int)g.target - sh.head, target_bytes = g.target >= sh.head ? (tv >> 2) * 16 : -1;
        const f4 off_target = {(tv & 3) == 0 ? g.c : 0.0f, (tv & 3) == 1 ? g.c : 0.0f, (tv & 3) == 2 ? g.c : 0.0f, (tv & 3) == 3 ? g.c : 0.0f};
        const int64_t single = part == 0 ? sh.single((int)threadIdx.x) : -1;
        if (single >= 0) {
            const float r = grad_at<EXTRA>(one, rm, ks, g);
            out[single] = single == g.target ? r - g.c : r;
        }
        const int next = next_live(row + stride);
        const float* xn = logits + (int64_t)(next < rows ? next : row) * cols;
        const RowShape shn(xn, cols);
        const SlotBuffer gs(out + sh.head, sh.n4), xs(xn + shn.head, next < rows ? shn.n4 : 0);   // (no slots: loads of nothing)
        int off = lane_bytes;
#pragma unroll
        for (int k = 0; k < kPartVpt; k++) {
            f4 r;
#pragma unroll
            for (int c = 0; c < 4; c++) r[c] = holds_exp(EXTRA) ? grad_of_exp<EXTRA>(v[k][c], ga, gb) : grad_at<EXTRA>(v[k][c], rm, ks, g);
            if (target_bytes == off) r -= off_target;
            gs.store<kNontemporal>(r, off);
            v[k] = xs.load<kNontemporal>(off);
            SERAPH_NEXT_SLOT(off);
        }
        listed = row;
        if (next >= rows) break;
        row = next;
        const int64_t c = part == 0 ? shn.single((int)threadIdx.x) : -1;
        one = c >= 0 ? xn[c] : -INFINITY;
    }
    if constexpr (Op::kList) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        write_entries(row, bcast.g, bcast.st.m);
    }
#undef SERAPH_NEXT_SLOT
}

static int shared_parts(int64_t cols) { return (int)ceil_div(ceil_div(cols / 4, kBlock), kPartVpt); }
static bool is_shared(int64_t cols) { return cols > 32768 && shared_parts(cols) <= kMaxParts; }
static inline size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }
static size_t shared_ws_bytes(int64_t rows, int64_t cols, int64_t top_k) {
    if (rows <= 0 || cols <= 0 || !is_shared(cols)) return 0;
    return up16((size_t)rows * sizeof(RowPrep)) + (size_t)rows * shared_parts(cols) * sizeof(PartRecord) + 2 * up16((size_t)rows * (size_t)(top_k > 0 ? top_k : 0) * 4);
}

static std::atomic<int> g_spin_limit{1 << 16};                    // waits of ~0.3 us each

template <class Op, int EXTRA>
static int launch_shared(const Op& op, const float* logits, float* grad, int64_t rows, int64_t cols, int64_t top_k, void* ws, hipStream_t st) {
    const int P = shared_parts(cols);
    char* p = reinterpret_cast<char*>(ws);
    RowPrep* prep = reinterpret_cast<RowPrep*>(p);
    PartRecord* records = reinterpret_cast<PartRecord*>(p += up16((size_t)rows * sizeof(RowPrep)));
    float* list_q = reinterpret_cast<float*>(p += (size_t)rows * P * sizeof(PartRecord));
    float* list_z = reinterpret_cast<float*>(p += up16((size_t)rows * (size_t)top_k * 4));
    const size_t lds = Op::kList ? list_bytes((int)top_k, hash_buckets((int)top_k)) : 0;
    const unsigned prep_grid = (unsigned)(Op::kList ? rows : ceil_div(rows, kPrepRows));
    hipLaunchKernelGGL((prepare_rows_kernel<Op>), dim3(prep_grid), dim3(64), lds, st, op, logits, rows, cols, P, prep, records, list_q, list_z);
    SERAPH_LAUNCH_CHECK();
    int64_t G = (int64_t)num_compute_units() * kPartsPerCu / P * P;
    if (G < P) G = P;
    if (G > rows * P) G = rows * P;
    hipLaunchKernelGGL((shared_rows_kernel<Op, EXTRA>), dim3((unsigned)G), dim3(kBlock), 0, st, op, logits, grad, (int)rows, cols, P, prep, records,
                       list_q, list_z, g_spin_limit.load(), grad == logits ? 1 : 0);
    SERAPH_LAUNCH_CHECK();
    return SERAPH_OK;
}

// ---------------------------------------------------------------- long rows read once
// Forward only (T = 1): nothing has to be held.  A row is cut into `splits` runs of vectors, each streamed by one workgroup whose
// waves keep a running reference value each and sums per lane; one wave per row then puts the runs' results together.
// Splitting serves few rows, which alone would leave most of the chip idle, and evens out the last round of many.  A row in
// one run (runs NULL) is finished by its own workgroup.
//
// The reference value is one for all lanes of a wave: the maximum of its first batch, until a logit exceeds it by kSlack, which is
// rare behind 2048 logits.  What the sums are multiplied by then, and where waves and runs are joined, is an exponential in 64
// bits (exp_below), so a logit takes one of the hardware's and no more.  The slack costs nothing in digits, as long as it is
// small: the argument of a logit above the reference is rounded as that of one as far below it.  (Without it, with 64-bit
// factors at every new maximum: 8 x 151936 in 12.1 us instead of 11.4; at 2, 3 and 4 it is 11.5, 11.4 and 11.5.)
constexpr float kSlack = 3.0f;

// Sums referred to another value m >= st.m.
struct WideSums { double s, x; };
template <int EXTRA>
__device__ __forceinline__ WideSums referred(RowStats st, float m) {
    static_assert(EXTRA == kNone || EXTRA == kEntropy, "at T = 1");
    const double d = (double)st.m - (double)m, r = exp_below(d);
    WideSums o{st.s == 0.0f ? 0.0 : (double)st.s * r, 0.0};
    if (EXTRA == kEntropy) o.x = st.s == 0.0f || r == 0.0 ? 0.0 : ((double)st.x + d * (double)st.s) * r;
    return o;
}
// The results that the lanes of a wave hold, put together.
template <int EXTRA>
__device__ __forceinline__ RowStats join_lanes(RowStats got) {
    const float m = wave_top(got.m);
    const WideSums o = referred<EXTRA>(got, m);
    return RowStats{m, (float)wave_total(o.s), EXTRA != kNone ? (float)wave_total(o.x) : 0.0f};
}

template <class Op, int EXTRA, int BLOCK>
__global__ __launch_bounds__(BLOCK) void streamed_rows_kernel(Op op, const float* logits, int64_t cols, int splits, RowStats* runs) {
    constexpr int kAhead = 8;                                     // vectors in flight per lane
    __shared__ RowStats waves[BLOCK / 64];
    const int64_t row = blockIdx.x / (unsigned)splits;
    const int run = (int)(blockIdx.x % (unsigned)splits);
    if (!op.live(row)) {
        if (run == 0 && threadIdx.x == 0) op.dead(row);
        return;
    }
    float zt = 0.0f;
    if (!runs && threadIdx.x == 0) zt = logits[row * cols + op.target(row)];
    const float* x = logits + row * cols;
    const RowShape sh(x, cols);
    const f4* xv = reinterpret_cast<const f4*>(x + sh.head);
    const int per_run = ((sh.n4 + splits - 1) / splits + BLOCK - 1) / BLOCK * BLOCK;
    const int first = run * per_run, end = first + per_run < sh.n4 ? first + per_run : sh.n4;
    const ExpScale ks = op.k;
    const int lane = (int)threadIdx.x & 63;
    RowStats st{kLowest, 0.0f, 0.0f};                             // m is the same for the whole wave
    auto refer_to = [&](float m) {                                // (every lane of the wave is here)
        if (!__any(m > st.m + kSlack)) return;
        m = wave_top(fmaxf(m, st.m));
        const WideSums o = referred<EXTRA>(st, m);
        st = RowStats{m, (float)o.s, (float)o.x};
    };
    auto take = [&](const f4 (&v)[kAhead]) {
        float m = kLowest;
#pragma unroll
        for (int j = 0; j < kAhead; j++) m = fmaxf(m, fmaxf(fmaxf(v[j].x, v[j].y), fmaxf(v[j].z, v[j].w)));
        refer_to(m);
        float s = 0.0f, ex = 0.0f;                                // a batch's own sums: the lane's take one addition of 32
#pragma unroll
        for (int j = 0; j < kAhead; j++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const float e = exp_of(v[j][c], st.m, ks);
                s += e;
                if (EXTRA != kNone) ex += extra_of<EXTRA>(v[j][c], st.m, e);
            }
        st.s += s;
        st.x += ex;
    };
    int base = __builtin_amdgcn_readfirstlane(first + (int)threadIdx.x - lane);      // the wave's first lane's vector
    for (; base + 63 + (kAhead - 1) * BLOCK < end; base += kAhead * BLOCK) {
        f4 v[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) v[j] = __builtin_nontemporal_load(xv + base + lane + j * BLOCK);
        __builtin_amdgcn_sched_barrier(0);                        // all loads first: else the scheduler waits for one to save registers
        take(v);
    }
    if (base < end) {                                             // the rest, in flight together as well
        f4 v[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            v[j] = f4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (base + lane + j * BLOCK < end) v[j] = __builtin_nontemporal_load(xv + base + lane + j * BLOCK);
        }
        take(v);
    }
    if (run == 0 && threadIdx.x < 64) {                           // the row's single values
        const int64_t single = sh.single(lane);
        const float z = single >= 0 ? x[single] : -INFINITY;
        refer_to(z);
        const float e = exp_of(z, st.m, ks);
        st.s += e;
        if (EXTRA != kNone) st.x += extra_of<EXTRA>(z, st.m, e);
    }
    st.s = wave_total(st.s);
    if (EXTRA != kNone) st.x = wave_total(st.x);
    if (lane == 0) waves[threadIdx.x >> 6] = st;
    __syncthreads();
    if (threadIdx.x >= 64) return;
    const RowStats o = join_lanes<EXTRA>(lane < BLOCK / 64 ? waves[lane] : RowStats{kLowest, 0.0f, 0.0f});
    if (lane == 0) {
        if (runs) runs[row * splits + run] = o;
        else op.template finish<EXTRA>(row, o, zt, ListSums{0.0, 0.0, 0.0f});
    }
}

template <class Op, int EXTRA>
__global__ __launch_bounds__(kBlock) void join_runs_kernel(Op op, const float* logits, int64_t rows, int64_t cols, int splits, const RowStats* runs) {
    const int64_t row = (int64_t)blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6);
    const int lane = (int)threadIdx.x & 63;
    if (row >= rows || !op.live(row)) return;
    const RowStats total = join_lanes<EXTRA>(lane < splits ? runs[row * splits + lane] : RowStats{kLowest, 0.0f, 0.0f});
    if (lane == 0) op.template finish<EXTRA>(row, total, logits[row * cols + op.target(row)], ListSums{0.0, 0.0, 0.0f});
}

constexpr int kMaxRuns = 64;
static int streamed_runs(int64_t rows, int64_t cols) {
    const int64_t wanted = ceil_div(8192, rows), most = cols / 4 / (8 * kBlock);      // a run has eight vectors per lane at least
    const int64_t n = wanted < most ? wanted : most;
    return (int)(n < 1 ? 1 : n > kMaxRuns ? kMaxRuns : n);
}
// Few rows, each short enough for one workgroup of 1024 lanes: one launch instead of two.  A row's exponentials take one CU about
// 5.2 us per 100000 columns, on top of the 3 us of any launch; a second launch costs the host 4 us, and little in a
// captured graph.  Whole / cut, us a call in a sequence of calls (in a graph):
//              32800 columns           50021                 98304                 151936                163840
//     1 row    7.4 / 12 (4.9 / 5.4)    7.3 / 12 (6.4 / 5.8)  7.8 / 12 (8.2 / 5.4)  11 / 12 (11 / 5.8)    11 / 12 (11 / 5.3)
//     8 rows   7.4 / 12 (5.3 / 6.2)    7.4 / 12 (6.8 / 6.4)  8.1 / 12 (8.3 / 5.9)  15 / 12 (14 / 7.0)    13 / 12 (14 / 6.0)
//    64 rows   7.5 / 12 (6.1 / 7.4)    8.3 / 12 (8.5 / 8.5)  11 / 12 (11 / 9.1)    17 / 13 (17 / 12)     16 / 12 (16 / 11)
//   128 rows   7.4 / 12 (6.8 / 8.7)    8.8 / 12 (9.0 / 10)   12 / 12 (12 / 13)     18 / 18 (18 / 18)     18 / 17 (18 / 17)
//   256 rows   8.2 / 12 (8.3 / 12)     11 / 14 (11 / 14)     18 / 19 (18 / 19)     26 / 30 (26 / 29)     28 / 29 (28 / 29)
// (8 rows of 151936 columns took 11.4 us in other buffers.)  So the limits give away up to 5 us at 8 to 64 rows of 151936 columns and
// more, and in graphs at few rows beyond 50000.
static bool in_one_run(int64_t rows, int64_t cols) { return rows <= 256 && cols <= 163840; }
static size_t streamed_ws_bytes(int64_t rows, int64_t cols) {
    return rows > 0 && cols > 32768 && !in_one_run(rows, cols) ? up16((size_t)rows * streamed_runs(rows, cols) * sizeof(RowStats)) : 0;
}

template <class Op, int EXTRA>
static int launch_runs(const Op& op, const float* logits, int64_t rows, int64_t cols, int splits, RowStats* runs, hipStream_t st) {
    if (in_one_run(rows, cols))
        hipLaunchKernelGGL((streamed_rows_kernel<Op, EXTRA, 1024>), dim3((unsigned)rows), dim3(1024), 0, st, op, logits, cols, 1, runs);
    else
        hipLaunchKernelGGL((streamed_rows_kernel<Op, EXTRA, kBlock>), dim3((unsigned)(rows * splits)), dim3(kBlock), 0, st, op, logits, cols, splits, runs);
    SERAPH_LAUNCH_CHECK();
    return SERAPH_OK;
}

template <class Op, int EXTRA>
static int launch_streamed(const Op& op, const float* logits, int64_t rows, int64_t cols, void* ws, hipStream_t st) {
    const int splits = streamed_runs(rows, cols);
    RowStats* runs = in_one_run(rows, cols) ? nullptr : reinterpret_cast<RowStats*>(ws);
    const int rc = launch_runs<Op, EXTRA>(op, logits, rows, cols, splits, runs, st);
    if (rc != SERAPH_OK || !runs) return rc;
    hipLaunchKernelGGL((join_runs_kernel<Op, EXTRA>), dim3((unsigned)ceil_div(rows, kBlock / 64)), dim3(kBlock), 0, st, op, logits, rows, cols, splits, runs);
    SERAPH_LAUNCH_CHECK();
    return SERAPH_OK;
}

// ---------------------------------------------------------------- rows swept from memory
// One workgroup per row: maximum, sums, gradient, each a sweep of its own, for rows beyond what kMaxParts workgroups hold
// (1245184 columns).
template <class Op, int EXTRA>
__global__ __launch_bounds__(kBlock) void swept_rows_kernel(Op op, const float* logits, float* grad, int64_t cols) {
    __shared__ float red[3][kBlock / 64];
    __shared__ RowGrad bcast;
    extern __shared__ char list_lds[];
    const int64_t row = blockIdx.x;
    float* out = grad + row * cols;
    if (!op.live(row)) {
        for (int64_t c = threadIdx.x; c < cols; c += kBlock) out[c] = 0.0f;
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
    ListRoom room{};
    ListSums sums{0.0, 0.0, 0.0f};
    if constexpr (Op::kList) {
        room = list_room(list_lds, op.list.top_k, hash_buckets(op.list.top_k));
        if (threadIdx.x < 64) sums = read_list(op.list, row, x, cols, op.inv_temp, op.k, room);
    }
    if (threadIdx.x == 0) {
        const int64_t t = op.target(row);
        bcast = op.template finish<EXTRA>(row, st, t >= 0 ? x[t] : 0.0f, sums);
    }
    __syncthreads();
    const RowGrad g = bcast;
    for (int64_t c = threadIdx.x; c < cols; c += kBlock) {
        const float v = grad_at<EXTRA>(x[c], st.m, k, g);
        out[c] = c == g.target ? v - g.c : v;
    }
    if constexpr (Op::kList) {
        const float es = op.entry_scale(row);
        __syncthreads();                                          // the sweep has written every entry's place
        for (int i = threadIdx.x; i < op.list.top_k; i += kBlock) {
            const uint32_t id = room.id[i];
            if (id != kNoId) out[id] = grad_at<EXTRA>(room.z[i], st.m, k, g) - es * room.q[i] - ((int64_t)id == g.target ? g.c : 0.0f);
        }
    }
}

template <class Op, int EXTRA>
static int launch_rows(const Op& op, const float* logits, float* grad, int64_t rows, int64_t cols, int64_t top_k, void* ws, hipStream_t st) {
    const size_t lds = Op::kList ? list_bytes((int)top_k, cols <= 32768 ? (int)cols / 4 + 2 : hash_buckets((int)top_k)) : 0;
    if (cols <= 32768) {
        const int64_t n4 = cols / 4;
#define HELD(B, V) hipLaunchKernelGGL((held_rows_kernel<Op, EXTRA, B, V>), dim3((unsigned)rows), dim3(B), lds, st, op, logits, grad, (int)cols)
        if (n4 <= 256) HELD(256, 1);
        else if (n4 <= 2 * 256) HELD(256, 2);
        else if (n4 <= 4 * 256) HELD(256, 4);
        else if (n4 <= 8 * 256) HELD(256, 8);
        else if (n4 <= 12 * 256) HELD(256, 12);
        else if (n4 <= 8 * 512) HELD(512, 8);
        else if (n4 <= 12 * 512) HELD(512, 12);
        else HELD(512, 16);
#undef HELD
        SERAPH_LAUNCH_CHECK();
        return SERAPH_OK;
    }
    if constexpr (Op::kGrad) {
        if (is_shared(cols)) return launch_shared<Op, EXTRA>(op, logits, grad, rows, cols, top_k, ws, st);
        hipLaunchKernelGGL((swept_rows_kernel<Op, EXTRA>), dim3((unsigned)rows), dim3(kBlock), lds, st, op, logits, grad, cols);
        SERAPH_LAUNCH_CHECK();
        return SERAPH_OK;
    } else {
        return launch_streamed<Op, EXTRA>(op, logits, rows, cols, ws, st);
    }
}

// ---------------------------------------------------------------- preference pairs
// Every row's factor follows from both sequences of its pair, so the logits are read twice: once for the rows' statistics,
// once for the gradient, which then is a streaming pass without any reduction.
struct PreferenceArgs {
    const float* logits;
    const uint32_t* targets;
    const float* ref_logp;
    const uint32_t* seq_starts;
    const RowStats* runs;          // `splits` results for each supervised row; where it is one, x is the target's logit
    float *loss_pairs, *scores, *logp_rows;
    int64_t rows, cols;
    int pairs, splits, kind, average;
    float beta, smoothing, margin;
};

// What the gradient pass needs of a row: its maximum, the factor of exp(z - m), and what the target takes off.
constexpr uint32_t kDead = 0xffffffffu;
struct RowFactor { float m, a, c; uint32_t target; };

struct PairRowsOp {
    static constexpr bool kGrad = false, kList = false;
    Supervision rows;
    RowStats* runs;
    RowFactor* factors;            // NULL: not wanted
    float* logp_rows;
    ExpScale k;
    __device__ __forceinline__ bool live(int64_t r) const { return rows.live(r); }
    __device__ __forceinline__ int64_t target(int64_t r) const { return rows.targets[r]; }
    __device__ __forceinline__ void dead(int64_t r) const {
        if (factors) factors[r] = RowFactor{0.0f, 0.0f, 0.0f, kDead};
        if (logp_rows) logp_rows[r] = 0.0f;
    }
    template <int EXTRA>
    __device__ __forceinline__ RowGrad finish(int64_t r, RowStats st, float zt, const ListSums&, bool = true) const {
        runs[r] = RowStats{st.m, st.s, zt};
        return RowGrad{0.0f, 0.0f, 0.0f, -1};
    }
};

// A row's runs put together, in their order and in 64 bits (exp_below); four loads in flight.
__device__ __forceinline__ RowStats joined(const PreferenceArgs& p, int64_t r) {
    const RowStats* runs = p.runs + r * p.splits;
    RowStats st = runs[0];
    double s = st.s;
    for (int i = 1; i < p.splits; i += 4) {
        RowStats o[4];
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = runs[i + j < p.splits ? i + j : 0];
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (i + j < p.splits) {
                const double f = exp_below(-fabs((double)o[j].m - (double)st.m));
                s = o[j].m > st.m ? fma(s, f, (double)o[j].s) : fma((double)o[j].s, f, s);
                st.m = fmaxf(st.m, o[j].m);
            }
    }
    st.s = (float)s;
    return st;
}
__device__ __forceinline__ RowFactor factor_of(RowStats st, uint32_t target, double f) {
    return RowFactor{st.m, (float)(-f / (double)st.s), (float)-f, target};
}

// The two sequences of a pair, their scores and its loss; slope0 and slope1 are d(mean loss) / d(log-probability of a token) of
// either side.  Called by a whole workgroup, half of which sums each side; sums in 64 bits and in one order whoever forms them.
// first, last, end: of this half's sequence; st: this lane's first row there
struct Pair { int64_t first, last, end; double slope0, slope1; RowStats st; };
template <int BLOCK>
__device__ __forceinline__ Pair read_pair(const PreferenceArgs& p, int pair, double (*red)[BLOCK / 64], bool writes) {
    Pair q;
    q.st = RowStats{0.0f, 1.0f, 0.0f};
    const int side = (int)threadIdx.x / (BLOCK / 2);
    const uint32_t* b = p.seq_starts + 2 * (int64_t)pair + side;
    q.first = b[0];
    q.end = b[1];
    q.last = q.end < p.rows ? q.end : p.rows;
    double sum = 0.0, n = 0.0;
    for (int64_t r = q.first + (int)threadIdx.x % (BLOCK / 2); r < q.last; r += BLOCK / 2) {
        const uint32_t t = p.targets[r];
        const RowStats st = joined(p, r);                         // (not yet known to hold anything: the loads of a row do not wait for each other)
        if (r < q.first + BLOCK / 2) q.st = st;
        const float ref = p.ref_logp ? p.ref_logp[r] : 0.0f;
        if ((int64_t)t >= p.cols || r + 1 >= q.end) continue;
        const float zt = p.splits == 1 ? st.x : p.logits[r * p.cols + t];
        const double logp = ((double)zt - (double)st.m) - log_of_sum(st.s);
        if (writes && p.logp_rows) p.logp_rows[r] = (float)logp;
        sum += logp - (double)ref;
        n += 1.0;
    }
    sum = wave_total(sum);
    n = wave_total(n);
    if ((threadIdx.x & 63) == 0) {
        red[0][threadIdx.x >> 6] = sum;
        red[1][threadIdx.x >> 6] = n;
    }
    __syncthreads();
    double score0 = 0.0, score1 = 0.0, count0 = 0.0, count1 = 0.0, loss;
#pragma unroll
    for (int w = 0; w < BLOCK / 128; w++) {
        score0 += red[0][w];
        count0 += red[1][w];
        score1 += red[0][w + BLOCK / 128];
        count1 += red[1][w + BLOCK / 128];
    }
    if (!p.average || count0 == 0.0) count0 = 1.0;
    if (!p.average || count1 == 0.0) count1 = 1.0;
    score0 /= count0;
    score1 /= count1;
    const double beta = (double)p.beta, gap = score0 - score1, h = beta * gap - (double)p.margin;
    double slope;                                                 // d loss / d gap
    if (p.kind == SERAPH_PREFERENCE_SIGMOID) {
        const double eps = (double)p.smoothing, soft = log1p(exp(-fabs(h)));
        loss = h != h ? h : 0.0;
        // (a term whose factor is 0 is left out: a gap is infinite where an answer holds a token that cannot be chosen)
        if (eps != 1.0) loss += (1.0 - eps) * (soft + fmax(-h, 0.0));
        if (eps != 0.0) loss += eps * (soft + fmax(h, 0.0));
        slope = beta * (eps - 1.0 / (1.0 + exp(h)));
    } else if (p.kind == SERAPH_PREFERENCE_HINGE) {
        loss = h >= 1.0 ? 0.0 : 1.0 - h;
        slope = h >= 1.0 ? 0.0 : h < 1.0 ? -beta : h;             // (NaN stays NaN)
    } else {
        const double d = gap - 0.5 / beta;
        loss = d * d;
        slope = 2.0 * d;
    }
    q.slope0 = slope / (double)p.pairs / count0;
    q.slope1 = -slope / (double)p.pairs / count1;
    if (writes && threadIdx.x == 0) {
        p.loss_pairs[pair] = (float)loss;
        if (p.scores) {
            p.scores[2 * (int64_t)pair] = (float)score0;
            p.scores[2 * (int64_t)pair + 1] = (float)score1;
        }
    }
    return q;
}

constexpr int kPairBlock = 512;

// One workgroup per pair writes the factors of its rows (those that are not supervised have been marked by the pass before).
__global__ __launch_bounds__(1024) void pair_kernel(PreferenceArgs p, RowFactor* factors) {
    __shared__ double red[2][1024 / 64];
    const Pair q = read_pair<1024>(p, (int)blockIdx.x, red, true);
    const double f = threadIdx.x < 512 ? q.slope0 : q.slope1;
    for (int64_t r = q.first + (int)threadIdx.x % 512; r < q.last; r += 512) {
        const uint32_t t = p.targets[r];
        if ((int64_t)t < p.cols && r + 1 < q.end) factors[r] = factor_of(r < q.first + 512 ? q.st : joined(p, r), t, f);
    }
}

// One vector per lane: of all shapes tried (1 to 16 vectors per lane, 128 to 1024 lanes, either order of the rows) the smallest
// pieces of work keep reads and writes best mixed: 4096 x 151936 in 0.80 ms (6.2 TB/s), with eight vectors 0.92 ms.
__device__ __forceinline__ void pair_grad(const PreferenceArgs& p, float* grad, int64_t row, int run, const RowFactor& f) {
    const float* x = p.logits + row * p.cols;
    float* out = grad + row * p.cols;
    const RowShape sh(x, p.cols);
    const int i4 = run * kPairBlock + (int)threadIdx.x;
    const int64_t single = run == 0 ? sh.single((int)threadIdx.x) : -1;
    f4a4* to = reinterpret_cast<f4a4*>(out + sh.head) + i4;
    if (f.target == kDead) {
        if (i4 < sh.n4) __builtin_nontemporal_store(f4a4{0, 0, 0, 0}, to);
        if (single >= 0) out[single] = 0.0f;
        return;
    }
    if (i4 < sh.n4) {
        const f4 v = __builtin_nontemporal_load(reinterpret_cast<const f4*>(x + sh.head) + i4);
        const int c = (int)f.target - (sh.head + i4 * 4);
        f4a4 r;
#pragma unroll
        for (int j = 0; j < 4; j++) r[j] = f.a * exp_of(v[j], f.m, kUnitScale) - (j == c ? f.c : 0.0f);
        __builtin_nontemporal_store(r, to);
    }
    if (single >= 0) out[single] = f.a * exp_of(x[single], f.m, kUnitScale) - (single == (int64_t)f.target ? f.c : 0.0f);
}

__global__ __launch_bounds__(kPairBlock) void pair_grad_kernel(PreferenceArgs p, float* grad, const RowFactor* factors, int splits_of_row, int64_t first_row) {
    const int64_t row = first_row + (int64_t)(blockIdx.x / (unsigned)splits_of_row);
    pair_grad(p, grad, row, (int)(blockIdx.x % (unsigned)splits_of_row), factors[row]);
}

// A batch whose gradient is a single round of workgroups: each reads its row's pair by itself, which takes less than the launch
// it replaces.  `pairs` further workgroups write the pairs' own results.  (In place too: the targets' logits have been
// kept by the pass before, and every other logit is read by the workgroup that overwrites it.)
__global__ __launch_bounds__(kPairBlock) void small_pairs_kernel(PreferenceArgs p, float* grad, int splits_of_row) {
    __shared__ double red[2][kPairBlock / 64];
    const int64_t row = (int64_t)(blockIdx.x / (unsigned)splits_of_row);
    const int run = (int)(blockIdx.x % (unsigned)splits_of_row);
    if (row >= p.rows) {
        read_pair<kPairBlock>(p, (int)(blockIdx.x - (unsigned)(p.rows * splits_of_row)), red, true);
        return;
    }
    RowFactor f{0.0f, 0.0f, 0.0f, kDead};
    const int sq = find_seq(p.seq_starts, 2 * p.pairs, row);
    const uint32_t t = p.targets[row];
    if (sq < 2 * p.pairs && row >= (int64_t)p.seq_starts[sq] && row + 1 < (int64_t)p.seq_starts[sq + 1] && (int64_t)t < p.cols) {
        const Pair q = read_pair<kPairBlock>(p, sq / 2, red, false);
        f = factor_of(joined(p, row), t, sq & 1 ? q.slope1 : q.slope0);
    }
    pair_grad(p, grad, row, run, f);
}

}  // namespace seraph

using namespace seraph;

#define REQUIRE_ROWS(op)                                                                                              \
    SERAPH_REQUIRE(rows > 0 && cols > 0 && rows <= kMaxRows && cols <= 0x7fffffff, op ": bad shape %lld x %lld",       \
                   (long long)rows, (long long)cols)
// A gradient that covers other logits than its own would overwrite what another workgroup still reads.
#define REQUIRE_GRAD(op)                                                                                              \
    SERAPH_REQUIRE(grad == logits || (uintptr_t)grad >= (uintptr_t)(logits + rows * cols) || (uintptr_t)logits >= (uintptr_t)(grad + rows * cols), \
                   op ": grad has to be the logits themselves or not overlap them")
#define REQUIRE_WS(op, need)                                                                                          \
    do {                                                                                                              \
        if ((need) && (!ws || ws_bytes < (need) || !aligned16(ws))) {                                                 \
            set_error(op ": scratch of %zu bytes, 16-byte aligned, needed (given %zu)", (size_t)(need), ws_bytes);     \
            return SERAPH_ERR_WORKSPACE;                                                                              \
        }                                                                                                             \
    } while (0)

namespace seraph {
// The buffers of a call (NULL and empty ones count for nothing).  What it writes shares memory with none of the others: every
// workgroup that works on a row reads the row's inputs, at times that nothing orders against another one's writes.
struct Extent { const void* at; size_t bytes; bool written; };
template <int N>
static bool apart(const Extent (&e)[N]) {
    for (int i = 0; i < N; i++) {
        if (!e[i].written || !e[i].at || !e[i].bytes) continue;
        const uintptr_t a = (uintptr_t)e[i].at;
        for (int j = 0; j < N; j++) {
            const uintptr_t b = (uintptr_t)e[j].at;
            if (j != i && b && a < b + e[j].bytes && b < a + e[i].bytes) return false;
        }
    }
    return true;
}
static size_t words(int64_t n) { return (size_t)n * 4; }
static size_t offsets_bytes(const uint32_t* seq_starts, int64_t batch) { return seq_starts ? words(batch + 1) : 0; }
// (a gradient in the logits' place is one buffer)
static size_t logits_bytes(const float* logits, const float* grad, int64_t rows, int64_t cols) { return logits == grad ? 0 : words(rows * cols); }
}  // namespace seraph
#define REQUIRE_APART(op, ...)                                                                                        \
    do {                                                                                                              \
        const Extent extents[] = {__VA_ARGS__};                                                                       \
        SERAPH_REQUIRE(apart(extents), op ": an output overlaps another buffer of the call");                         \
    } while (0)

extern "C" {

void seraph_objectives_exchange_spins(int spins) {
    if (spins >= 0) g_spin_limit = spins;
}

size_t seraph_token_logprobs_ws_bytes(int64_t rows, int64_t cols) { return streamed_ws_bytes(rows, cols); }

int seraph_token_logprobs(const float* logits, const uint32_t* targets, float* logp, float* lse, float* entropy,
                          const uint32_t* seq_starts, int batch, int64_t rows, int64_t cols,
                          void* ws, size_t ws_bytes, seraph_stream_t s) {
    if (rows == 0 || cols == 0) return SERAPH_OK;
    REQUIRE_ROWS("token_logprobs");
    SERAPH_REQUIRE(logits && targets && logp, "token_logprobs: NULL pointer");
    SERAPH_REQUIRE(!seq_starts || batch >= 1, "token_logprobs: packed call needs batch >= 1");
    REQUIRE_WS("token_logprobs", seraph_token_logprobs_ws_bytes(rows, cols));
    REQUIRE_APART("token_logprobs", {logits, words(rows * cols), false}, {targets, words(rows), false}, {seq_starts, offsets_bytes(seq_starts, batch), false},
                  {logp, words(rows), true}, {lse, words(rows), true}, {entropy, words(rows), true},
                  {ws, seraph_token_logprobs_ws_bytes(rows, cols), true});
    LogprobsOp op{{targets, nullptr, seq_starts, batch, cols}, logp, lse, entropy, kUnitScale};
    if (entropy) return launch_rows<LogprobsOp, kEntropy>(op, logits, nullptr, rows, cols, 0, ws, as_stream(s));
    return launch_rows<LogprobsOp, kNone>(op, logits, nullptr, rows, cols, 0, ws, as_stream(s));
}

size_t seraph_policy_grad_ws_bytes(int64_t rows, int64_t cols) { return shared_ws_bytes(rows, cols, 0); }

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
    REQUIRE_GRAD("policy_grad");
    REQUIRE_WS("policy_grad", seraph_policy_grad_ws_bytes(rows, cols));
    REQUIRE_APART("policy_grad", {logits, logits_bytes(logits, grad, rows, cols), false}, {actions, words(rows), false}, {advantages, words(rows), false},
                  {old_logp, words(rows), false}, {ref_logp, words(rows), false}, {weights, words(rows), false},
                  {seq_starts, offsets_bytes(seq_starts, batch), false}, {grad, words(rows * cols), true}, {loss_rows, words(rows), true},
                  {logp_rows, words(rows), true}, {kl_rows, words(rows), true}, {entropy_rows, words(rows), true},
                  {ws, seraph_policy_grad_ws_bytes(rows, cols), true});
    const float scale = valid_rows > 0 ? 1.0f / (float)valid_rows : 0.0f;
    PolicyOp op{{actions, weights, seq_starts, batch, cols}, advantages, old_logp, ref_logp, loss_rows, logp_rows, kl_rows, entropy_rows,
                options->clip_low, options->clip_high, options->kl_coef, options->entropy_coef, scale, kUnitScale};
    if (options->entropy_coef != 0.0f || entropy_rows) return launch_rows<PolicyOp, kEntropy>(op, logits, grad, rows, cols, 0, ws, as_stream(s));
    return launch_rows<PolicyOp, kNone>(op, logits, grad, rows, cols, 0, ws, as_stream(s));
}

static int pair_runs(int64_t rows, int64_t cols) { return cols <= 32768 || in_one_run(rows, cols) ? 1 : streamed_runs(rows, cols); }
size_t seraph_preference_grad_ws_bytes(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0) return 0;
    return up16((size_t)rows * sizeof(RowFactor)) + up16((size_t)rows * pair_runs(rows, cols) * sizeof(RowStats));
}

int seraph_preference_grad(const float* logits, const uint32_t* targets, const float* ref_logp, float* grad,
                           float* loss_pairs, float* scores, float* logp_rows, const seraph_preference_options_t* options,
                           const uint32_t* seq_starts, int pairs, int64_t rows, int64_t cols,
                           void* ws, size_t ws_bytes, seraph_stream_t s) {
    if (rows == 0 || cols == 0) return SERAPH_OK;
    REQUIRE_ROWS("preference_grad");
    SERAPH_REQUIRE(logits && targets && grad && loss_pairs && options && seq_starts, "preference_grad: NULL pointer");
    SERAPH_REQUIRE(pairs > 0 && pairs <= 0x3fffff, "preference_grad: bad number of pairs %d", pairs);
    SERAPH_REQUIRE(options->kind >= SERAPH_PREFERENCE_SIGMOID && options->kind <= SERAPH_PREFERENCE_SQUARED, "preference_grad: unknown loss %d", options->kind);
    SERAPH_REQUIRE(isfinite(options->beta) && options->beta > 0.0f, "preference_grad: beta %g must be positive", (double)options->beta);
    SERAPH_REQUIRE(options->label_smoothing >= 0.0f && options->label_smoothing <= 1.0f, "preference_grad: label smoothing %g outside [0, 1]", (double)options->label_smoothing);
    SERAPH_REQUIRE(isfinite(options->margin), "preference_grad: margin must be finite");
    REQUIRE_GRAD("preference_grad");
    REQUIRE_WS("preference_grad", seraph_preference_grad_ws_bytes(rows, cols));
    REQUIRE_APART("preference_grad", {logits, logits_bytes(logits, grad, rows, cols), false}, {targets, words(rows), false}, {ref_logp, words(rows), false},
                  {seq_starts, offsets_bytes(seq_starts, 2 * (int64_t)pairs), false}, {grad, words(rows * cols), true}, {loss_pairs, words(pairs), true},
                  {scores, words(2 * (int64_t)pairs), true}, {logp_rows, words(rows), true}, {ws, seraph_preference_grad_ws_bytes(rows, cols), true});
    hipStream_t st = as_stream(s);
    const int splits = pair_runs(rows, cols);
    RowFactor* factors = reinterpret_cast<RowFactor*>(ws);
    RowStats* runs = reinterpret_cast<RowStats*>(reinterpret_cast<char*>(ws) + up16((size_t)rows * sizeof(RowFactor)));
    const int64_t row_splits = ceil_div(ceil_div(cols, 4), kPairBlock);
    const bool small = splits == 1 && rows * row_splits + pairs <= 4 * (int64_t)num_compute_units();      // four workgroups of 512 lanes on a CU
    PairRowsOp op{{targets, nullptr, seq_starts, 2 * pairs, cols}, runs, small ? nullptr : factors, logp_rows, kUnitScale};
    const int rc = cols <= 32768 ? launch_rows<PairRowsOp, kNone>(op, logits, nullptr, rows, cols, 0, nullptr, st)
                                 : launch_runs<PairRowsOp, kNone>(op, logits, rows, cols, splits, splits == 1 ? nullptr : runs, st);
    if (rc != SERAPH_OK) return rc;
    const PreferenceArgs a{logits, targets, ref_logp, seq_starts, runs, loss_pairs, scores, logp_rows, rows, cols, pairs, splits,
                           options->kind, options->average, options->beta, options->label_smoothing, options->margin};
    if (small) {
        hipLaunchKernelGGL(small_pairs_kernel, dim3((unsigned)(rows * row_splits + pairs)), dim3(kPairBlock), 0, st, a, grad, (int)row_splits);
        SERAPH_LAUNCH_CHECK();
        return SERAPH_OK;
    }
    hipLaunchKernelGGL(pair_kernel, dim3((unsigned)pairs), dim3(1024), 0, st, a, factors);
    SERAPH_LAUNCH_CHECK();
    const int64_t at_once = 0x7fffff / row_splits;                // less than 2^32 lanes in a launch: beyond 64 GB of logits one more
    for (int64_t first = 0; first < rows; first += at_once) {
        const int64_t n = rows - first < at_once ? rows - first : at_once;
        hipLaunchKernelGGL(pair_grad_kernel, dim3((unsigned)(n * row_splits)), dim3(kPairBlock), 0, st, a, grad, factors, (int)row_splits, first);
        SERAPH_LAUNCH_CHECK();
    }
    return SERAPH_OK;
}

size_t seraph_distill_grad_ws_bytes(int64_t rows, int64_t cols, int64_t top_k) { return shared_ws_bytes(rows, cols, top_k); }

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
    REQUIRE_GRAD("distill_grad");
    REQUIRE_WS("distill_grad", seraph_distill_grad_ws_bytes(rows, cols, top_k));
    REQUIRE_APART("distill_grad", {logits, logits_bytes(logits, grad, rows, cols), false}, {teacher_ids, words(rows * top_k), false},
                  {teacher_logits, words(rows * top_k) / (options->teacher_type == SERAPH_TYPE_F32 ? 1 : 2), false}, {teacher_lse, words(rows), false},
                  {targets, words(rows), false}, {weights, words(rows), false}, {seq_starts, offsets_bytes(seq_starts, batch), false},
                  {grad, words(rows * cols), true}, {loss_rows, words(rows), true}, {ws, seraph_distill_grad_ws_bytes(rows, cols, top_k), true});
    const float scale = valid_rows > 0 ? 1.0f / (float)valid_rows : 0.0f;
    if (options->soft_coef == 0.0f) top_k = 0;                    // the list is not read: 0 times what it holds need not be 0
    DistillOp op{{nullptr, weights, seq_starts, batch, cols}, {teacher_ids, teacher_logits, teacher_lse, options->teacher_type, (int)top_k},
                 targets, loss_rows, options->soft_coef, options->hard_coef, scale, ExpScale::of(1.0 / (double)options->temperature), 1.0 / (double)options->temperature};
    // At T = 1 the two parts share their exponentials, at T = 2 one is the other's square; any other T takes two for each logit.  T = 1,
    // 2 and 1.5: 98.6, 99.4 and 105.4 us at 2047 x 32000 with 256 listed, 867, 872 and 894 us at 4096 x 151936 with 64.
    if (options->hard_coef != 0.0f && options->temperature == 2.0f) return launch_rows<DistillOp, kSquare>(op, logits, grad, rows, cols, top_k, ws, as_stream(s));
    if (options->hard_coef != 0.0f && options->temperature != 1.0f) return launch_rows<DistillOp, kSecond>(op, logits, grad, rows, cols, top_k, ws, as_stream(s));
    return launch_rows<DistillOp, kNone>(op, logits, grad, rows, cols, top_k, ws, as_stream(s));
}

}  // extern "C"
