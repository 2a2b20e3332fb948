// Verification of drafted tokens (kvmem_hip_verify_draft): row by row of a
// request, draft x stays where u q(x) < p(x), p = softmax(logits / temperature);
// the next token is drawn from max(p - q, 0) at the first refusal, else from the
// last row's p.
//
// Every logit is read once: bytes bound it for many rows, three short dependent
// launches for few.
//   parts    a workgroup per part of a row: the part's maximum (with its lowest
//            id) and sum of exponentials relative to it
//   decide   a workgroup per request: joins its rows' parts, tests its drafts in
//            order, and draws the next token wherever p alone decides it, from the
//            part sums first and then inside the one part that holds the border
//   rest     where a refused draft had probabilities, the parts' sums of
//            max(p - q, 0), then the draw from those
// Exponentials and sums are fp64: a draw compares a running sum with u times the
// total, and of 10^5 ids' borders fp32 sums would misplace one in a few hundred
// draws; fp64 ones none in 10^8.
#include "kvmem_internal.hpp"

#include <algorithm>
#include <cmath>

#include "recurrent.hpp"

namespace kvmem_hip {

constexpr uint32_t kVerifyThreads = 256;
constexpr uint32_t kVerifyMaxDraft = 127;
constexpr int kVerifyWide = 4;  // groups of 8 ids a thread, in parts for many rows
constexpr uint32_t kVerifyFull = 8192;  // parts of many rows
constexpr uint32_t kVerifyMaxVocab = 1u << 24;

struct Part {
    double sum;   // of exp((logit - max) / temperature); 0: nothing above -inf
    float max;    // largest logit
    uint32_t at;  // its lowest id
};

// What a request's draw needs from the decide kernel.
struct Choice {
    double scale;   // 1 / sum of the row's exponentials
    float max;      // the row's largest logit
    uint32_t row;   // of the refused draft
    uint32_t pending;  // the draw is from max(p - q, 0)
    uint32_t pad[3];
};

struct VerifyParams {
    const uint8_t *logits;
    const uint8_t *probs;
    uint64_t logits_nb, probs_nb;
    int type, probs_type;
    uint32_t n_vocab, n_rows, n_seq, max_draft;
    const uint32_t *q_start;
    const int32_t *tokens;
    const float *temperature;
    const float *u_accept;
    const float *u_sample;
    const uint32_t *kv_len;
    int32_t *tokens_out;
    uint32_t *n_accepted;
    uint32_t *n_keep;
    uint32_t *kv_len_out;
    uint32_t part;       // ids of a part
    uint32_t n_parts;    // of a row
    bool vec, probs_vec; // 16-byte aligned rows
    Part *parts;         // [n_seq][max_draft + 1][n_parts]
    double *rest;        // [n_seq][n_parts]
    Choice *choice;      // [n_seq]
};

// Rows of request s: first, and how many are looked at.
__device__ inline uint32_t rows_of(const VerifyParams &p, uint32_t s, uint32_t &count, uint32_t &all) {
    const uint32_t most = p.max_draft + 1;
    const uint64_t first = p.q_start ? p.q_start[s] : static_cast<uint64_t>(s) * most;
    uint64_t end = p.q_start ? p.q_start[s + 1] : first + most;
    all = end > first ? static_cast<uint32_t>(end - first) : 0u;
    end = end < p.n_rows ? end : p.n_rows;
    count = end > first ? static_cast<uint32_t>(end - first) : 0u;
    count = count < most ? count : most;
    return static_cast<uint32_t>(first);
}

__device__ inline float load_float(const uint8_t *p, int type, uint64_t i) {
    if (type == KVMEM_TYPE_F32) {
        return reinterpret_cast<const float *>(p)[i];
    }
    const uint16_t h = reinterpret_cast<const uint16_t *>(p)[i];
    return type == KVMEM_TYPE_F16 ? static_cast<float>(__builtin_bit_cast(_Float16, h))
                                  : __uint_as_float(static_cast<uint32_t>(h) << 16);
}

template <typename T>
__device__ inline void load_eight_of(const uint8_t *row, bool vec, uint32_t v, uint32_t end, float (&x)[8]) {
    if (vec && v % 8 == 0 && v + 8 <= end) {
        RawRow<T, 8> raw;
        load_raw<T, 8>(row + static_cast<uint64_t>(v) * sizeof(T), raw);
        widen<T, 8>(raw, x);
        return;
    }
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) {
        x[e] = static_cast<float>(reinterpret_cast<const T *>(row)[v + e < end ? v + e : end - 1]);
    }
}

// Ids v..v+7 of a row (v < end; ids at or beyond `end` repeat the one before it).
__device__ inline void load_eight(const uint8_t *row, int type, bool vec, uint32_t v, uint32_t end, float (&x)[8]) {
    if (type == KVMEM_TYPE_F32) {
        load_eight_of<float>(row, vec, v, end, x);
    } else if (type == KVMEM_TYPE_F16) {
        load_eight_of<_Float16>(row, vec, v, end, x);
    } else {
        load_eight_of<__bf16>(row, vec, v, end, x);
    }
}

// A logit: NaN counts as -inf.
__device__ inline float load_logit(const uint8_t *p, int type, uint64_t i) {
    const float x = load_float(p, type, i);
    return x == x ? x : -INFINITY;
}

// exp((x - max) / temperature) for x <= max, inv = 1 / temperature, in fp64: with
// n = rint(32 t / ln 2), e^t = 2^(n / 32) e^r, |r| <= ln 2 / 64, where e^r's series
// to r^5 leaves 2e-15 and 2^(n mod 32 / 32) comes from a table in LDS (its 32 entries
// fill the 64 banks once: lanes never collide).  t is cut at -800, whose weight is 0;
// that is also where -inf and NaN end.  Thirteen fp64 operations against some 40 of the
// library's exp, which has to hold for every argument.
struct ExpTable {
    double entry[32];
};
__device__ inline void fill_table(ExpTable &t) {
    if (threadIdx.x < 32) {
        t.entry[threadIdx.x] = exp2(static_cast<double>(threadIdx.x) / 32.0);
    }
    __syncthreads();
}
__device__ inline double weight_of(const ExpTable &table, float x, double inv, double max_inv) {
    const double t = fmax(__builtin_fma(static_cast<double>(x), inv, -max_inv), -800.0);
    constexpr double magic = 0x1.8p52;  // leaves n in the low bits
    const double k = __builtin_fma(t, 0x1.71547652b82fep+5, magic);
    const int n = static_cast<int>(__builtin_bit_cast(uint64_t, k));
    const double r = __builtin_fma(k - magic, -0x1.62e42fefa39efp-6, t);
    double e = __builtin_fma(r, 1.0 / 120.0, 1.0 / 24.0);
    e = __builtin_fma(r, e, 1.0 / 6.0);
    e = __builtin_fma(r, e, 0.5);
    e = __builtin_fma(r, e, 1.0);
    e = __builtin_fma(r, e, 1.0);
    return __builtin_ldexp(e * table.entry[n & 31], n >> 5);
}

__device__ inline bool better(float m, uint32_t at, float m2, uint32_t at2) {
    return m > m2 || (m == m2 && at < at2);
}

// Sum over the workgroup, in an order that never changes; every thread has it.
__device__ inline double block_sum(double v, double *lds) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        v += __shfl_xor(v, m, 64);
    }
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) {
        lds[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

__device__ inline void block_best(float &m, uint32_t &at, float *lds_m, uint32_t *lds_at) {
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const float m2 = __shfl_xor(m, x, 64);
        const uint32_t at2 = __shfl_xor(at, x, 64);
        if (better(m2, at2, m, at)) {
            m = m2, at = at2;
        }
    }
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) {
        lds_m[threadIdx.x >> 6] = m;
        lds_at[threadIdx.x >> 6] = at;
    }
    __syncthreads();
    m = lds_m[0], at = lds_at[0];
    for (int i = 1; i < 4; ++i) {
        if (better(lds_m[i], lds_at[i], m, at)) {
            m = lds_m[i], at = lds_at[i];
        }
    }
}

__device__ inline double inv_temperature(const VerifyParams &p, uint32_t s, bool &greedy) {
    const float t = p.temperature ? p.temperature[s] : 1.0f;
    greedy = !(t > 0.0f);
    return greedy ? 1.0 : 1.0 / static_cast<double>(t);
}

// A thread's numbers of a part: groups of 8 (16 bytes of a 16-bit row, 32 of an F32
// one), the workgroup's side by side.  `first` is the part's first id, ids at or beyond
// `end` are -inf.
template <typename T, int GROUPS, bool VEC>
__device__ inline void load_part(const uint8_t *row, uint32_t first, uint32_t end, float (&x)[GROUPS][8]) {
#pragma unroll
    for (uint32_t j = 0; j < GROUPS; ++j) {
        const uint32_t v = first + (j * kVerifyThreads + threadIdx.x) * 8u;
        if (VEC && v + 8 <= end) {
            RawRow<T, 8> raw;
            load_raw<T, 8>(row + static_cast<uint64_t>(v) * sizeof(T), raw);
            widen<T, 8>(raw, x[j]);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                x[j][i] = v + i < end ? static_cast<float>(reinterpret_cast<const T *>(row)[v + i]) : -INFINITY;
            }
        }
    }
}

template <typename T, int GROUPS, bool VEC>
__global__ __launch_bounds__(kVerifyThreads) void verify_parts_kernel(const VerifyParams p) {
    __shared__ ExpTable table;
    __shared__ double lds_d[4];
    __shared__ float lds_m[4];
    __shared__ uint32_t lds_at[4];
    const uint32_t s = blockIdx.z, i = blockIdx.y, part = blockIdx.x;
    uint32_t count, all;
    const uint32_t first = rows_of(p, s, count, all);
    if (i >= count) {
        return;
    }
    const uint8_t *row = p.logits + (static_cast<uint64_t>(first) + i) * p.logits_nb;
    constexpr uint32_t ids = GROUPS * 8 * kVerifyThreads;
    const uint32_t v0 = part * ids, v1 = p.n_vocab - v0 < ids ? p.n_vocab : v0 + ids;
    float x[GROUPS][8];
    load_part<T, GROUPS, VEC>(row, v0, v1, x);
    fill_table(table);
    bool greedy;
    const double inv = inv_temperature(p, s, greedy);
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            m = __builtin_fmaxf(m, x[j][e]);  // NaN is left out
        }
    }
#pragma unroll
    for (int e = 1; e < 64; e <<= 1) {
        m = __builtin_fmaxf(m, __shfl_xor(m, e, 64));
    }
    if ((threadIdx.x & 63u) == 0) {
        lds_m[threadIdx.x >> 6] = m;
    }
    __syncthreads();
    m = __builtin_fmaxf(__builtin_fmaxf(lds_m[0], lds_m[1]), __builtin_fmaxf(lds_m[2], lds_m[3]));
    double sum = 0.0;
    uint32_t at = 0xffffffffu;
    if (greedy || m == INFINITY) {
        if (m > -INFINITY) {
#pragma unroll
            for (int j = GROUPS - 1; j >= 0; --j) {
#pragma unroll
                for (int e = 7; e >= 0; --e) {
                    at = x[j][e] == m ? v0 + (static_cast<uint32_t>(j) * kVerifyThreads + threadIdx.x) * 8u +
                                            static_cast<uint32_t>(e)
                                      : at;
                }
            }
            float mine = at == 0xffffffffu ? -INFINITY : m;
            block_best(mine, at, lds_m, lds_at);
        }
    } else if (m > -INFINITY) {
        const double max_inv = static_cast<double>(m) * inv;
        double part_sum[2] = {};
#pragma unroll
        for (int j = 0; j < GROUPS; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                part_sum[e & 1] += weight_of(table, x[j][e], inv, max_inv);
            }
        }
        sum = block_sum(part_sum[0] + part_sum[1], lds_d);
    }
    if (threadIdx.x == 0) {
        p.parts[(static_cast<uint64_t>(s) * (p.max_draft + 1) + i) * p.n_parts + part] = Part{sum, m, at};
    }
}

// Sum over ids [a, b) of a part of the weights that `weight` makes of a logit and (where
// probs are given) a probability; eight are read at a time.
template <typename F>
__device__ inline double sum_ids(const VerifyParams &p, const uint8_t *logits, const uint8_t *probs, uint32_t v0,
                                 uint32_t a, uint32_t b, F weight) {
    double sum = 0.0;
    for (; a < b; a += 8) {
        float x[8], q[8];
        load_eight(logits, p.type, p.vec, v0 + a, v0 + b, x);
        if (probs) {
            load_eight(probs, p.probs_type, p.probs_vec, v0 + a, v0 + b, q);
        }
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            sum += a + e < b ? weight(v0 + a + e, x[e], probs ? q[e] : 0.0f) : 0.0;
        }
    }
    return sum;
}

struct PickLds {
    double sum[4];
    double before;
    uint32_t found[4], fallback[4];
};

// Running sum over the wave's lanes, this lane's included.
__device__ inline double wave_scan(double v) {
    const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const double y = __shfl_up(v, x, 64);
        v += lane >= static_cast<uint32_t>(x) ? y : 0.0;
    }
    return v;
}

// The first of n weights whose running sum (from `start`) passes `target`, by the whole
// workgroup; `before` is the running sum in front of it.  Where none passes, the last
// positive one (n if there is none).  Threads sum runs of `per` weights (sum_of(first,
// end)), running sums of the runs find one run, and its weights' (w) running sums the
// place in it (per <= 64).
template <typename S, typename W>
__device__ inline uint32_t block_pick(uint32_t n, uint32_t per, double start, double target, S sum_of, W w,
                                      PickLds &lds, double &before) {
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
    const uint32_t a = min(n, threadIdx.x * per);
    const double sum = sum_of(a, min(n, a + per));
    const bool some = sum > 0.0;
    double run = wave_scan(sum);
    __syncthreads();
    if (lane == 63) {
        lds.sum[wave] = run;
    }
    __syncthreads();
    double base = start;
    for (uint32_t i = 0; i < wave; ++i) {
        base += lds.sum[i];
    }
    run += base;
    const uint64_t passed = __ballot(some && run > target), there = __ballot(some);
    if (lane == 0) {
        lds.found[wave] = passed ? wave * 64u + static_cast<uint32_t>(__builtin_ctzll(passed)) : kVerifyThreads;
        lds.fallback[wave] = there ? wave * 64u + 63u - static_cast<uint32_t>(__builtin_clzll(there)) : kVerifyThreads;
    }
    __syncthreads();
    uint32_t owner = kVerifyThreads;
    for (int i = 3; i >= 0; --i) {
        owner = lds.found[i] < kVerifyThreads ? lds.found[i] : owner;
    }
    for (int i = 3; i >= 0 && owner == kVerifyThreads; --i) {
        owner = lds.fallback[i];
    }
    if (owner == kVerifyThreads) {
        before = start;
        return n;  // nothing positive
    }
    if (threadIdx.x == owner) {
        lds.before = run - sum;
    }
    __syncthreads();
    const double front = lds.before;
    if (per == 1) {
        before = front;
        __syncthreads();
        return owner;
    }
    // every wave finds the same place
    const uint32_t i = owner * per + lane;
    const double mine = lane < per && i < n ? w(i) : 0.0;
    const double upto = front + wave_scan(mine);
    const uint64_t over = __ballot(mine > 0.0 && upto > target), positive = __ballot(mine > 0.0);
    const int at = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(positive | 1u);
    before = __shfl(upto - mine, at, 64);
    __syncthreads();
    return owner * per + static_cast<uint32_t>(at);
}

struct Row {
    double sum;
    float max;
    uint32_t at;
};

// A row's parts together, by one wave.
__device__ inline Row join_row(const VerifyParams &p, const ExpTable &table, const Part *parts, double inv) {
    const uint32_t lane = threadIdx.x & 63u;
    float m = -INFINITY;
    uint32_t at = 0xffffffffu;
    for (uint32_t i = lane; i < p.n_parts; i += 64) {
        const Part x = parts[i];
        if (better(x.max, x.at, m, at)) {
            m = x.max, at = x.at;
        }
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const float m2 = __shfl_xor(m, x, 64);
        const uint32_t at2 = __shfl_xor(at, x, 64);
        if (better(m2, at2, m, at)) {
            m = m2, at = at2;
        }
    }
    double sum = 0.0;
    for (uint32_t i = lane; i < p.n_parts; i += 64) {
        const Part x = parts[i];
        sum += x.sum > 0.0 ? x.sum * weight_of(table, x.max, inv, static_cast<double>(m) * inv) : 0.0;
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        sum += __shfl_xor(sum, x, 64);
    }
    return Row{sum, m, at};
}

__device__ inline void write_request(const VerifyParams &p, uint32_t s, uint32_t first, uint32_t count, uint32_t all,
                                     uint32_t accepted) {
    int32_t *out = p.tokens_out + static_cast<uint64_t>(s) * (p.max_draft + 1);
    for (uint32_t i = threadIdx.x; i <= p.max_draft; i += kVerifyThreads) {
        out[i] = i < accepted ? p.tokens[first + i + 1] : -1;
    }
    if (threadIdx.x == 0) {
        const uint32_t keep = count ? accepted + 1 : 0u;
        p.n_accepted[s] = accepted;
        if (p.n_keep) {
            p.n_keep[s] = keep;
        }
        if (p.kv_len_out) {
            p.kv_len_out[s] = p.kv_len[s] - all + keep;
        }
    }
}

__device__ inline void write_token(const VerifyParams &p, uint32_t s, uint32_t accepted, uint32_t id) {
    if (threadIdx.x == 0) {
        p.tokens_out[static_cast<uint64_t>(s) * (p.max_draft + 1) + accepted] = static_cast<int32_t>(id);
    }
}

__global__ __launch_bounds__(kVerifyThreads) void verify_decide_kernel(const VerifyParams p) {
    __shared__ Row rows[kVerifyMaxDraft + 1];
    __shared__ uint8_t stays[kVerifyMaxDraft + 1];
    __shared__ PickLds lds;
    __shared__ double lds_d[4];
    __shared__ ExpTable table;
    fill_table(table);
    const uint32_t s = blockIdx.x;
    uint32_t count, all;
    const uint32_t first = rows_of(p, s, count, all);
    bool greedy;
    const double inv = inv_temperature(p, s, greedy);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (uint32_t i = wave; i < count; i += kVerifyThreads / 64) {
        const uint64_t r = static_cast<uint64_t>(first) + i;
        const Row row =
            join_row(p, table, p.parts + (static_cast<uint64_t>(s) * (p.max_draft + 1) + i) * p.n_parts, inv);
        if ((threadIdx.x & 63u) == 0) {
            rows[i] = row;
            bool ok = false;
            if (i + 1 < count) {
                const uint32_t x = static_cast<uint32_t>(p.tokens[r + 1]);
                if (x < p.n_vocab && row.max > -INFINITY) {
                    if (greedy || row.max == INFINITY) {
                        ok = x == row.at;
                    } else {
                        const double e =
                            weight_of(table, load_logit(p.logits + r * p.logits_nb, p.type, x), inv,
                                      static_cast<double>(row.max) * inv) /
                            row.sum;
                        const double q =
                            p.probs ? static_cast<double>(load_float(p.probs + r * p.probs_nb, p.probs_type, x)) : 1.0;
                        ok = static_cast<double>(p.u_accept[r]) * q < e;
                    }
                }
            }
            stays[i] = ok;
        }
    }
    __syncthreads();
    uint32_t accepted = 0;
    while (accepted + 1 < count && stays[accepted]) {
        ++accepted;
    }
    write_request(p, s, first, count, all, accepted);
    __syncthreads();  // tokens_out[accepted] is written again below
    if (threadIdx.x == 0) {
        p.choice[s].pending = 0;
    }
    if (count == 0) {
        return;
    }
    const Row row = rows[accepted];
    if (row.max == -INFINITY) {
        return;  // nothing to draw from: -1
    }
    if (greedy || row.max == INFINITY) {
        write_token(p, s, accepted, row.at);
        return;
    }
    const uint64_t r = static_cast<uint64_t>(first) + accepted;
    const bool refused = accepted + 1 < count;
    if (refused && p.probs) {
        if (threadIdx.x == 0) {
            p.choice[s] = Choice{1.0 / row.sum, row.max, accepted, 1u, {}};
        }
        return;
    }
    // the draw from p, without the refused draft
    const double max_inv = static_cast<double>(row.max) * inv;
    const Part *parts = p.parts + (static_cast<uint64_t>(s) * (p.max_draft + 1) + accepted) * p.n_parts;
    const uint8_t *logits = p.logits + r * p.logits_nb;
    uint32_t without = refused ? static_cast<uint32_t>(p.tokens[r + 1]) : 0xffffffffu;
    without = without < p.n_vocab ? without : 0xffffffffu;
    uint32_t cut = 0xffffffffu;  // its part, and that part's sum without it
    double cut_sum = 0.0;
    double total = row.sum;
    auto id_weight = [&](uint32_t v, float x, float) {
        return v == without ? 0.0 : weight_of(table, x, inv, max_inv);
    };
    auto part_weight = [&](uint32_t i) {
        const Part x = parts[i];
        return i == cut ? cut_sum : x.sum > 0.0 ? x.sum * weight_of(table, x.max, inv, max_inv) : 0.0;
    };
    auto parts_sum = [&](uint32_t a, uint32_t b) {
        double sum = 0.0;
        for (; a < b; ++a) {
            sum += part_weight(a);
        }
        return sum;
    };
    if (without != 0xffffffffu) {
        cut = without / p.part;
        const uint32_t v0 = cut * p.part, ids = min(p.part, p.n_vocab - v0), per = p.part / kVerifyThreads;
        const uint32_t a = min(ids, threadIdx.x * per);
        cut_sum = block_sum(sum_ids(p, logits, nullptr, v0, a, min(ids, a + per), id_weight), lds_d);
        total = 0.0;
        for (uint32_t i = threadIdx.x; i < p.n_parts; i += kVerifyThreads) {
            total += part_weight(i);
        }
        total = block_sum(total, lds_d);
        if (!(total > 0.0)) {  // the draft was all there is
            without = cut = 0xffffffffu;
            total = row.sum;
        }
    }
    const double target = static_cast<double>(p.u_sample[s]) * total;
    double before;
    const uint32_t part = block_pick(p.n_parts, (p.n_parts + kVerifyThreads - 1) / kVerifyThreads, 0.0, target,
                                     parts_sum, part_weight, lds, before);
    if (part >= p.n_parts) {
        return;
    }
    const uint32_t v0 = part * p.part;
    const uint32_t at = block_pick(
        min(p.part, p.n_vocab - v0), p.part / kVerifyThreads, before, target,
        [&](uint32_t a, uint32_t b) { return sum_ids(p, logits, nullptr, v0, a, b, id_weight); },
        [&](uint32_t i) { return id_weight(v0 + i, load_float(logits, p.type, v0 + i), 0.0f); }, lds, before);
    write_token(p, s, accepted, v0 + at);
}

__device__ inline double rest_of(const ExpTable &table, double scale, float logit, float q, double inv,
                                 double max_inv) {
    const double e = weight_of(table, logit, inv, max_inv) * scale - static_cast<double>(q);
    return e > 0.0 ? e : 0.0;
}

template <typename T, typename Q, int GROUPS, bool VEC>
__global__ __launch_bounds__(kVerifyThreads) void verify_rest_kernel(const VerifyParams p) {
    __shared__ ExpTable table;
    __shared__ double lds_d[4];
    const uint32_t s = blockIdx.y, part = blockIdx.x;
    const Choice c = p.choice[s];
    if (!c.pending) {
        return;
    }
    uint32_t count, all;
    const uint64_t r = static_cast<uint64_t>(rows_of(p, s, count, all)) + c.row;
    constexpr uint32_t ids = GROUPS * 8 * kVerifyThreads;
    const uint32_t v0 = part * ids, v1 = p.n_vocab - v0 < ids ? p.n_vocab : v0 + ids;
    float x[GROUPS][8], q[GROUPS][8];
    load_part<T, GROUPS, VEC>(p.logits + r * p.logits_nb, v0, v1, x);
    load_part<Q, GROUPS, VEC>(p.probs + r * p.probs_nb, v0, v1, q);
    fill_table(table);
    bool greedy;
    const double inv = inv_temperature(p, s, greedy);
    const double max_inv = static_cast<double>(c.max) * inv;
    double sum = 0.0;
#pragma unroll
    for (uint32_t j = 0; j < GROUPS; ++j) {
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            // behind the part's end logit and q are -inf
            sum += v0 + (j * kVerifyThreads + threadIdx.x) * 8u + e < v1
                       ? rest_of(table, c.scale, x[j][e], q[j][e], inv, max_inv)
                       : 0.0;
        }
    }
    sum = block_sum(sum, lds_d);
    if (threadIdx.x == 0) {
        p.rest[static_cast<uint64_t>(s) * p.n_parts + part] = sum;
    }
}

__global__ __launch_bounds__(kVerifyThreads) void verify_draw_kernel(const VerifyParams p) {
    __shared__ PickLds lds;
    __shared__ double lds_d[4];
    __shared__ ExpTable table;
    fill_table(table);
    const uint32_t s = blockIdx.x;
    const Choice c = p.choice[s];
    if (!c.pending) {
        return;
    }
    uint32_t count, all;
    const uint64_t r = static_cast<uint64_t>(rows_of(p, s, count, all)) + c.row;
    bool greedy;
    const double inv = inv_temperature(p, s, greedy);
    const uint8_t *logits = p.logits + r * p.logits_nb, *probs = p.probs + r * p.probs_nb;
    const double *rest = p.rest + static_cast<uint64_t>(s) * p.n_parts;
    const Part *parts = p.parts + (static_cast<uint64_t>(s) * (p.max_draft + 1) + c.row) * p.n_parts;
    const double max_inv = static_cast<double>(c.max) * inv;
    double total = 0.0;
    for (uint32_t i = threadIdx.x; i < p.n_parts; i += kVerifyThreads) {
        total += rest[i];
    }
    total = block_sum(total, lds_d);
    const bool left = total > 0.0;  // else p itself
    if (!left) {
        total = 1.0 / c.scale;
    }
    const double target = static_cast<double>(p.u_sample[s]) * total;
    double before;
    auto part_weight = [&](uint32_t i) {
        const Part x = parts[i];
        return left ? rest[i] : x.sum > 0.0 ? x.sum * weight_of(table, x.max, inv, max_inv) : 0.0;
    };
    const uint32_t part = block_pick(
        p.n_parts, (p.n_parts + kVerifyThreads - 1) / kVerifyThreads, 0.0, target,
        [&](uint32_t a, uint32_t b) {
            double sum = 0.0;
            for (; a < b; ++a) {
                sum += part_weight(a);
            }
            return sum;
        },
        part_weight, lds, before);
    if (part >= p.n_parts) {
        return;
    }
    const uint32_t v0 = part * p.part;
    auto id_weight = [&](uint32_t, float x, float q) {
        return left ? rest_of(table, c.scale, x, q, inv, max_inv) : weight_of(table, x, inv, max_inv);
    };
    const uint32_t at = block_pick(
        min(p.part, p.n_vocab - v0), p.part / kVerifyThreads, before, target,
        [&](uint32_t a, uint32_t b) { return sum_ids(p, logits, probs, v0, a, b, id_weight); },
        [&](uint32_t i) {
            return id_weight(v0 + i, load_float(logits, p.type, v0 + i), load_float(probs, p.probs_type, v0 + i));
        },
        lds, before);
    write_token(p, s, c.row, v0 + at);
}

template <typename T, int GROUPS>
static void launch_parts(hipStream_t stream, const VerifyParams &p) {
    const dim3 grid(p.n_parts, p.max_draft + 1, p.n_seq);
    if (p.vec) {
        verify_parts_kernel<T, GROUPS, true><<<grid, kVerifyThreads, 0, stream>>>(p);
    } else {
        verify_parts_kernel<T, GROUPS, false><<<grid, kVerifyThreads, 0, stream>>>(p);
    }
}

template <typename T, typename Q, int GROUPS>
static void launch_rest_groups(hipStream_t stream, const VerifyParams &p) {
    const dim3 grid(p.n_parts, p.n_seq);
    if (p.vec && p.probs_vec) {
        verify_rest_kernel<T, Q, GROUPS, true><<<grid, kVerifyThreads, 0, stream>>>(p);
    } else {
        verify_rest_kernel<T, Q, GROUPS, false><<<grid, kVerifyThreads, 0, stream>>>(p);
    }
}

template <typename T>
static void launch_rest(hipStream_t stream, const VerifyParams &p) {
    const bool wide = p.part == 8u * kVerifyWide * kVerifyThreads;
    if (p.probs_type == KVMEM_TYPE_F32) {
        wide ? launch_rest_groups<T, float, kVerifyWide>(stream, p) : launch_rest_groups<T, float, 1>(stream, p);
    } else if (p.probs_type == KVMEM_TYPE_F16) {
        wide ? launch_rest_groups<T, _Float16, kVerifyWide>(stream, p) : launch_rest_groups<T, _Float16, 1>(stream, p);
    } else {
        wide ? launch_rest_groups<T, __bf16, kVerifyWide>(stream, p) : launch_rest_groups<T, __bf16, 1>(stream, p);
    }
}

template <typename T>
static void launch_verify(hipStream_t stream, const VerifyParams &p) {
    if (p.part == 8u * kVerifyWide * kVerifyThreads) {
        launch_parts<T, kVerifyWide>(stream, p);
    } else {
        launch_parts<T, 1>(stream, p);
    }
    if (hipPeekAtLastError() != hipSuccess) {
        return;  // parts that were not written must not be read
    }
    verify_decide_kernel<<<p.n_seq, kVerifyThreads, 0, stream>>>(p);
    if (p.probs && p.max_draft && hipPeekAtLastError() == hipSuccess) {
        launch_rest<T>(stream, p);
        if (hipPeekAtLastError() == hipSuccess) {
            verify_draw_kernel<<<p.n_seq, kVerifyThreads, 0, stream>>>(p);
        }
    }
}

bool load_verify_kernels() {
    return load_kernel_object(&verify_decide_kernel);
}

struct VerifyPlan {
    uint32_t part, n_parts;
    size_t parts_bytes, rest_bytes, choice_bytes;
};

static VerifyPlan plan_verify(const kvmem_hip_verify_args *a) {
    VerifyPlan pl;
    const uint64_t logits = static_cast<uint64_t>(a->n_seq) * (a->max_draft + 1) * a->n_vocab;
    const uint32_t wide = 8u * kVerifyWide * kVerifyThreads;
    pl.part = logits / wide >= kVerifyFull || a->n_vocab > (1u << 21) ? wide : 8u * kVerifyThreads;
    pl.n_parts = (a->n_vocab + pl.part - 1) / pl.part;
    const size_t rows = static_cast<size_t>(a->n_seq) * (a->max_draft + 1);
    pl.parts_bytes = rows * pl.n_parts * sizeof(Part);
    pl.rest_bytes = (static_cast<size_t>(a->n_seq) * pl.n_parts * sizeof(double) + 15) / 16 * 16;
    pl.choice_bytes = a->n_seq * sizeof(Choice);
    return pl;
}

static const char *check_verify(const kvmem_hip_verify_args *a, int &code) {
    code = KVMEM_HIP_ERR_INVALID;
    if (!a) {
        return "verify_draft: null arguments";
    }
    if (!float_type_ok(a->type) || (a->probs && !float_type_ok(a->probs_type))) {
        code = KVMEM_HIP_ERR_UNSUPPORTED;
        return "verify_draft: logits and probs must be F32, F16 or BF16";
    }
    if (a->n_seq > 65535 || a->max_draft > kVerifyMaxDraft || a->n_vocab > kVerifyMaxVocab) {
        code = KVMEM_HIP_ERR_UNSUPPORTED;
        return "verify_draft: at most 65535 requests, 127 drafts, 2^24 ids";
    }
    if (a->n_vocab == 0) {
        return "verify_draft: no ids";
    }
    if (a->n_seq == 0) {
        code = KVMEM_HIP_OK;
        return nullptr;
    }
    if (!a->logits || !a->tokens || !a->u_accept || !a->u_sample || !a->tokens_out || !a->n_accepted) {
        return "verify_draft: null array";
    }
    if ((a->kv_len == nullptr) != (a->kv_len_out == nullptr)) {
        return "verify_draft: kv_len and kv_len_out go together";
    }
    const uintptr_t words = reinterpret_cast<uintptr_t>(a->q_start) | reinterpret_cast<uintptr_t>(a->tokens) |
                            reinterpret_cast<uintptr_t>(a->temperature) | reinterpret_cast<uintptr_t>(a->u_accept) |
                            reinterpret_cast<uintptr_t>(a->u_sample) | reinterpret_cast<uintptr_t>(a->kv_len) |
                            reinterpret_cast<uintptr_t>(a->tokens_out) | reinterpret_cast<uintptr_t>(a->n_accepted) |
                            reinterpret_cast<uintptr_t>(a->n_keep) | reinterpret_cast<uintptr_t>(a->kv_len_out);
    const uintptr_t at = reinterpret_cast<uintptr_t>(a->logits) | a->logits_nb;
    const uintptr_t probs_at = a->probs ? reinterpret_cast<uintptr_t>(a->probs) | a->probs_nb : 0;
    if (words % 4 || at % float_type_size(a->type) || (a->probs && probs_at % float_type_size(a->probs_type))) {
        return "verify_draft: arrays and rows must be aligned to their elements";
    }
    if (a->tokens_out == a->tokens) {
        return "verify_draft: outputs must not overlap inputs";
    }
    code = KVMEM_HIP_OK;
    return nullptr;
}

}  // namespace kvmem_hip

using namespace kvmem_hip;

extern "C" {

size_t kvmem_hip_verify_draft_workspace(const kvmem_hip_verify_args *a) {
    int code = 0;
    if (check_verify(a, code) || a->n_seq == 0) {
        return 0;
    }
    const VerifyPlan pl = plan_verify(a);
    return pl.parts_bytes + pl.rest_bytes + pl.choice_bytes;
}

int kvmem_hip_verify_draft(kvmem_hip_ctx *ctx, const kvmem_hip_verify_args *a) {
    if (!ctx) {
        return KVMEM_HIP_ERR_INVALID;
    }
    int code = 0;
    if (const char *why = check_verify(a, code)) {
        return fail(ctx, code, why);
    }
    if (a->n_seq == 0) {
        return KVMEM_HIP_OK;
    }
    const VerifyPlan pl = plan_verify(a);
    // a dispatch counts its work items in 32 bits
    if (static_cast<uint64_t>(pl.n_parts) * (a->max_draft + 1) * a->n_seq * kVerifyThreads >= uint64_t{1} << 32) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "verify_draft: too many rows for one launch");
    }
    VerifyParams p{};
    p.logits = static_cast<const uint8_t *>(a->logits);
    p.probs = static_cast<const uint8_t *>(a->probs);
    p.logits_nb = a->logits_nb;
    p.probs_nb = a->probs_nb;
    p.type = a->type;
    p.probs_type = a->probs_type;
    p.n_vocab = a->n_vocab;
    p.n_rows = a->n_rows;
    p.n_seq = a->n_seq;
    p.max_draft = a->max_draft;
    p.q_start = a->q_start;
    p.tokens = a->tokens;
    p.temperature = a->temperature;
    p.u_accept = a->u_accept;
    p.u_sample = a->u_sample;
    p.kv_len = a->kv_len;
    p.tokens_out = a->tokens_out;
    p.n_accepted = a->n_accepted;
    p.n_keep = a->n_keep;
    p.kv_len_out = a->kv_len_out;
    p.part = pl.part;
    p.n_parts = pl.n_parts;
    p.vec = ((reinterpret_cast<uintptr_t>(a->logits) | a->logits_nb) & 15u) == 0;
    p.probs_vec = ((reinterpret_cast<uintptr_t>(a->probs) | a->probs_nb) & 15u) == 0;
    (void) hipSetDevice(ctx->device);
    uint8_t *ws = nullptr;
    if (const int rc = call_workspace(ctx, ctx->verify_scratch, a->workspace, a->workspace_bytes,
                                      pl.parts_bytes + pl.rest_bytes + pl.choice_bytes, "verify_draft", &ws)) {
        return rc;
    }
    p.parts = reinterpret_cast<Part *>(ws);
    p.rest = reinterpret_cast<double *>(ws + pl.parts_bytes);
    p.choice = reinterpret_cast<Choice *>(ws + pl.parts_bytes + pl.rest_bytes);
    if (injected_fail(ctx, KVMEM_HIP_FAIL_LAUNCH, "verify_draft launch")) {
        return KVMEM_HIP_ERR_RUNTIME;
    }
    if (a->type == KVMEM_TYPE_F32) {
        launch_verify<float>(ctx->stream, p);
    } else if (a->type == KVMEM_TYPE_F16) {
        launch_verify<_Float16>(ctx->stream, p);
    } else {
        launch_verify<__bf16>(ctx->stream, p);
    }
    return hip_ok(ctx, hipGetLastError(), "verify_draft launch") ? KVMEM_HIP_OK : KVMEM_HIP_ERR_RUNTIME;
}

}  // extern "C"
