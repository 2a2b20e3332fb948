// Verification of drafted tokens (kvmem_hip_verify_draft): row by row of a
// request, draft x stays where u q(x) < p(x), p = softmax(logits / temperature);
// the next token is drawn from max(p - q, 0) at the first refusal, else from the
// last row's p.
//
//   parts    a workgroup per 2048 ids of a row: their maximum (with its lowest id) and
//            the sum of exponentials relative to it: every logit, once
//   decide   a workgroup per request: joins its rows' parts, tests its drafts in
//            order, and draws the next token wherever p alone decides it, from the
//            part sums first and then inside the one part that holds the border (read
//            again, as are the drafts' logits and the part of a draft left out)
//   rest     where a refused draft had probabilities, the parts' sums of
//            max(p - q, 0): its row's logits again, and
//   draw     the draw from those (the border's part once more)
// Exponentials and sums are fp64: a draw compares a running sum with u times the
// total, and of 10^5 ids' borders fp32 sums would misplace one in a few hundred
// draws; a relative error of 10^-13, one in 10^7.
#include "kvmem_internal.hpp"

#include <algorithm>
#include <cmath>

#include "recurrent.hpp"

namespace kvmem_hip {

constexpr uint32_t kVerifyThreads = 256;
constexpr uint32_t kVerifyMaxDraft = 127;
constexpr uint32_t kPartIds = 8 * kVerifyThreads;
// Parts from which a wave takes a whole one.  Rows of 152000 ids, by four waves / by one:
// 64 rows (4800 parts) 25.8 / 25.3 us, 32 rows 21.5 / 21.9, 8 rows 16.6 / 18.2.
constexpr uint64_t kManyParts = 4096;
constexpr uint32_t kVerifyMaxVocab = 1u << 24;

constexpr uint32_t kNowhere = 0xffffffffu;

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
    uint32_t n_parts;    // of a row
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

// exp((x - max) / temperature) for x <= max, inv = 1 / temperature, in fp64, the
// difference first: it is 0 at the maximum and rounded once elsewhere, however small the
// temperature (max / temperature, rounded by itself, is off by 2^-53 of its size).  With
// n = rint(256 t / ln 2), e^t = 2^(n / 256) e^r, |r| <= ln 2 / 512, where e^r's series
// to r^3 leaves 1.4e-13 and 2^(n mod 256 / 256) comes from a table in LDS.  t is cut at
// -800, whose weight is 0; that is also where -inf and NaN end.  Twelve fp64 operations
// (a table of 32, to r^5: fourteen, 5 % of the largest calls) against some 40 of the
// library's exp, which has to hold for every argument.
__constant__ double kExpCoarse[16] = {
    0x1.0000000000000p+0, 0x1.0b5586cf9890fp+0, 0x1.172b83c7d517bp+0, 0x1.2387a6e756238p+0,
    0x1.306fe0a31b715p+0, 0x1.3dea64c123422p+0, 0x1.4bfdad5362a27p+0, 0x1.5ab07dd485429p+0,
    0x1.6a09e667f3bcdp+0, 0x1.7a11473eb0187p+0, 0x1.8ace5422aa0dbp+0, 0x1.9c49182a3f090p+0,
    0x1.ae89f995ad3adp+0, 0x1.c199bdd85529cp+0, 0x1.d5818dcfba487p+0, 0x1.ea4afa2a490dap+0,
};  // 2^(i / 16)
__constant__ double kExpFine[16] = {
    0x1.0000000000000p+0, 0x1.00b1afa5abcbfp+0, 0x1.0163da9fb3335p+0, 0x1.02168143b0281p+0,
    0x1.02c9a3e778061p+0, 0x1.037d42e11bbccp+0, 0x1.04315e86e7f85p+0, 0x1.04e5f72f654b1p+0,
    0x1.059b0d3158574p+0, 0x1.0650a0e3c1f89p+0, 0x1.0706b29ddf6dep+0, 0x1.07bd42b72a836p+0,
    0x1.0874518759bc8p+0, 0x1.092bdf66607e0p+0, 0x1.09e3ecac6f383p+0, 0x1.0a9c79b1f3919p+0,
};  // 2^(i / 256)
struct ExpTable {
    double entry[256];
};
template <uint32_t THREADS = kVerifyThreads> __device__ inline void fill_table(ExpTable &t) {
#pragma unroll
    for (uint32_t i = threadIdx.x; i < 256; i += THREADS) {
        t.entry[i] = kExpCoarse[i >> 4] * kExpFine[i & 15u];
    }
    __syncthreads();
}
__device__ inline double weight_of(const ExpTable &table, float x, double inv, double max) {
    const double t = fmax((static_cast<double>(x) - max) * inv, -800.0);
    constexpr double magic = 0x1.8p52;  // leaves n in the low bits
    const double k = __builtin_fma(t, 0x1.71547652b82fep+8, magic);
    const int n = static_cast<int>(__builtin_bit_cast(uint64_t, k));
    const double r = __builtin_fma(k - magic, -0x1.62e42fefa39efp-9, t);
    double e = __builtin_fma(r, 1.0 / 6.0, 0.5);
    e = __builtin_fma(r, e, 1.0);
    e = __builtin_fma(r, e, 1.0);
    return __builtin_ldexp(e * table.entry[n & 255], n >> 8);
}

// A wave's numbers combined by moves inside its rows of 16 lanes, then of lane 15 and
// 31 to the rows behind them: six steps of the VALU, where a lane permute a step would
// wait for LDS each time.  Lane 63 ends with all of them.  Lanes that a step has nothing
// for get `none`.
template <int CTRL, int ROWS> __device__ inline uint32_t moved(uint32_t none, uint32_t v) {
    return static_cast<uint32_t>(
        __builtin_amdgcn_update_dpp(static_cast<int>(none), static_cast<int>(v), CTRL, ROWS, 0xF, false));
}
template <int CTRL, int ROWS> __device__ inline double moved_or_zero(double v) {
    const uint64_t x = __builtin_bit_cast(uint64_t, v);
    const uint64_t hi = moved<CTRL, ROWS>(0u, static_cast<uint32_t>(x >> 32));
    return __builtin_bit_cast(double, hi << 32 | moved<CTRL, ROWS>(0u, static_cast<uint32_t>(x)));
}
constexpr int kRowShr = 0x110, kRowBcast15 = 0x142, kRowBcast31 = 0x143;

// Running sum over the wave's lanes, this lane's included.
__device__ inline double wave_scan(double v) {
    v += moved_or_zero<kRowShr + 1, 0xF>(v);
    v += moved_or_zero<kRowShr + 2, 0xF>(v);
    v += moved_or_zero<kRowShr + 4, 0xF>(v);
    v += moved_or_zero<kRowShr + 8, 0xF>(v);
    v += moved_or_zero<kRowBcast15, 0xA>(v);
    return v + moved_or_zero<kRowBcast31, 0xC>(v);
}
__device__ inline double wave_sum(double v) {
    const uint64_t x = __builtin_bit_cast(uint64_t, wave_scan(v));
    const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x >> 32), 63));
    return __builtin_bit_cast(double,
                              hi << 32 | static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), 63)));
}
template <int CTRL, int ROWS> __device__ inline float max_moved(float v) {
    return __builtin_fmaxf(v, __uint_as_float(moved<CTRL, ROWS>(__float_as_uint(v), __float_as_uint(v))));
}
__device__ inline float wave_max(float v) {
    v = max_moved<kRowShr + 1, 0xF>(v);
    v = max_moved<kRowShr + 2, 0xF>(v);
    v = max_moved<kRowShr + 4, 0xF>(v);
    v = max_moved<kRowShr + 8, 0xF>(v);
    v = max_moved<kRowBcast15, 0xA>(v);
    v = max_moved<kRowBcast31, 0xC>(v);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
template <int CTRL, int ROWS> __device__ inline uint32_t min_moved(uint32_t v) {
    return min(v, moved<CTRL, ROWS>(v, v));
}
__device__ inline uint32_t wave_min(uint32_t v) {
    v = min_moved<kRowShr + 1, 0xF>(v);
    v = min_moved<kRowShr + 2, 0xF>(v);
    v = min_moved<kRowShr + 4, 0xF>(v);
    v = min_moved<kRowShr + 8, 0xF>(v);
    v = min_moved<kRowBcast15, 0xA>(v);
    v = min_moved<kRowBcast31, 0xC>(v);
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}

// Over the workgroup, in an order that never changes; every thread has it.
__device__ inline double block_sum(double v, double *lds) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) {
        lds[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

__device__ inline double inv_temperature(const VerifyParams &p, uint32_t s, bool &greedy) {
    const float t = p.temperature ? p.temperature[s] : 1.0f;
    greedy = !(t > 0.0f);
    return greedy ? 1.0 : 1.0 / static_cast<double>(t);
}

// Eight neighbouring elements of a row, which may begin at any element: the card loads
// 16 bytes from any address.
template <typename T> __device__ inline void load_eight(const uint8_t *p, float (&x)[8]) {
    typedef T vec_t __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    const vec_t v = *reinterpret_cast<const vec_t *>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = static_cast<float>(v[i]);
    }
}

// A thread's eight numbers of a part (16 bytes of a 16-bit row, 32 of an F32 one).
// `first` is the part's first id, ids at or beyond `end` are -inf.
template <typename T>
__device__ inline void load_part(const uint8_t *row, uint32_t first, uint32_t end, float (&x)[8]) {
    const uint32_t v = first + threadIdx.x * 8u;
    if (v + 8 <= end) {
        load_eight<T>(row + static_cast<uint64_t>(v) * sizeof(T), x);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            x[i] = v + i < end ? static_cast<float>(reinterpret_cast<const T *>(row)[v + i]) : -INFINITY;
        }
    }
}

// A thread has GROUPS groups of eight ids.  Each wave sums relative to its own maximum,
// and the first joins them.  Bound by vector instructions, thirteen fp64 ones and two more
// an id and some ninety a wave to combine its lanes: with four groups a wave takes the
// whole part and combines a quarter as often.  512 rows of 152000 bf16 ids, the whole
// call: 80.1 us with one group, 73.6 with two, 68.0 with four (this kernel 49 us, 3.2
// TB/s); 8 rows of 32000 ids: 14.1, 14.9, 15.7.
template <typename T, int GROUPS>
__global__ __launch_bounds__(kVerifyThreads / GROUPS) void verify_parts_kernel(const VerifyParams p) {
    constexpr uint32_t waves = 4 / GROUPS, threads = kVerifyThreads / GROUPS;
    __shared__ ExpTable table;
    __shared__ Part of_waves[waves];
    const uint32_t s = blockIdx.z, i = blockIdx.y, v0 = blockIdx.x * kPartIds;
    uint32_t count, all;
    const uint32_t first = rows_of(p, s, count, all);
    if (i >= count) {
        return;
    }
    const uint8_t *row = p.logits + (static_cast<uint64_t>(first) + i) * p.logits_nb;
    float x[GROUPS][8];
#pragma unroll
    for (uint32_t j = 0; j < GROUPS; ++j) {
        load_part<T>(row, v0 + j * threads * 8u, p.n_vocab, x[j]);
    }
    fill_table<threads>(table);
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
    m = wave_max(m);
    double sum = 0.0;
    uint32_t at = kNowhere;
    if (greedy || m == INFINITY) {
#pragma unroll
        for (int j = GROUPS - 1; j >= 0; --j) {
#pragma unroll
            for (int e = 7; e >= 0; --e) {
                at = x[j][e] == m ? v0 + (static_cast<uint32_t>(j) * threads + threadIdx.x) * 8u +
                                        static_cast<uint32_t>(e)
                                  : at;
            }
        }
        at = wave_min(m > -INFINITY ? at : kNowhere);
    } else if (m > -INFINITY) {
        const double max = m;
        double part_sum[2] = {};
#pragma unroll
        for (int j = 0; j < GROUPS; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                part_sum[e & 1] += weight_of(table, x[j][e], inv, max);
            }
        }
        sum = wave_sum(part_sum[0] + part_sum[1]);
    }
    if constexpr (waves > 1) {
        if ((threadIdx.x & 63u) == 0) {
            of_waves[threadIdx.x >> 6] = Part{sum, m, at};
        }
        __syncthreads();
        if (threadIdx.x >= 64) {
            return;
        }
        const Part w = of_waves[threadIdx.x % waves];
        m = wave_max(w.max);
        at = wave_min(w.max == m ? w.at : kNowhere);
        sum = threadIdx.x < waves && w.sum > 0.0 && m < INFINITY
                  ? w.sum * weight_of(table, w.max, inv, static_cast<double>(m))
                  : 0.0;
        sum = wave_sum(sum);
    }
    if (threadIdx.x == 0) {
        p.parts[(static_cast<uint64_t>(s) * (p.max_draft + 1) + i) * p.n_parts + blockIdx.x] = Part{sum, m, at};
    }
}

struct PickLds {
    double sum[4];
    uint32_t first[4], last[4];
    double before;
    uint32_t part;
};

// The first thread whose running sum (from `start`) passes the target; where none does,
// the last with a positive sum (kNowhere if there is none).  `front` is the running sum
// before this thread.  The target is `target` times the sum of all with OF_ALL.
template <bool OF_ALL>
__device__ inline uint32_t block_find(double sum, double start, double &target, PickLds &lds, double &front) {
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
    double run = wave_scan(sum);
    if (lane == 63) {
        lds.sum[wave] = run;
    }
    __syncthreads();
    double all = start;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        run += i == wave ? all : 0.0;
        all += lds.sum[i];
    }
    if (OF_ALL) {
        target *= all;
    }
    const uint64_t there = __ballot(sum > 0.0), passed = __ballot(sum > 0.0 && run > target);
    if (lane == 0) {
        lds.first[wave] = passed ? wave * 64u + static_cast<uint32_t>(__builtin_ctzll(passed)) : kNowhere;
        lds.last[wave] = there ? wave * 64u + 64u - static_cast<uint32_t>(__builtin_clzll(there)) : 0u;
    }
    __syncthreads();
    const uint32_t first = min(min(lds.first[0], lds.first[1]), min(lds.first[2], lds.first[3]));
    const uint32_t last = max(max(lds.last[0], lds.last[1]), max(lds.last[2], lds.last[3]));  // and one
    front = run - sum;
    return first != kNowhere ? first : last - 1u;
}

// The part a draw ends in (kNowhere: nothing is positive), `target` turned from a
// fraction of the parts' weights into a running sum, `before` the one in front of the
// part.
template <typename W>
__device__ inline uint32_t pick_part(uint32_t n_parts, double &target, W weight, PickLds &lds, double &before) {
    const uint32_t per = (n_parts + kVerifyThreads - 1) / kVerifyThreads, a = threadIdx.x * per;
    double sum = 0.0;
    for (uint32_t i = a; i < min(n_parts, a + per); ++i) {
        sum += weight(i);
    }
    double front;
    const uint32_t at = block_find<true>(sum, 0.0, target, lds, front);
    if (at == threadIdx.x) {
        // of several parts, the first that passes, else the last positive one
        uint32_t part = a;
        double run = front;
        before = front;
        for (uint32_t i = a; per > 1 && i < min(n_parts, a + per); ++i) {
            const double w = weight(i);
            if (w > 0.0) {
                part = i;
                before = run;
                run += w;
                if (run > target) {
                    break;
                }
            }
        }
        lds.part = part;
        lds.before = before;
    }
    __syncthreads();
    before = lds.before;
    return at == kNowhere ? kNowhere : lds.part;
}

// The id a draw ends in, in a part of which this thread has the weights w[i] of ids
// v0 + threadIdx.x * 8 + i; its thread writes it.
__device__ inline void pick_id(uint32_t v0, double before, double target, const double (&w)[8], PickLds &lds,
                               int32_t *token) {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        sum += w[i];
    }
    double front;
    if (block_find<false>(sum, before, target, lds, front) != threadIdx.x) {
        return;
    }
    uint32_t found = 0;
    bool over = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        front += w[i];
        found = w[i] > 0.0 && !over ? static_cast<uint32_t>(i) : found;
        over = over || (w[i] > 0.0 && front > target);
    }
    *token = static_cast<int32_t>(v0 + threadIdx.x * 8u + found);
}

struct Row {
    double sum;
    float max;
    uint32_t at;
};

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

constexpr int kRowsAtOnce = 2;   // of a wave's rows, so that their loads and sums overlap
constexpr int kPartsHeld = 2;    // parts a lane keeps of a row; it reads others twice

template <typename T>
__global__ __launch_bounds__(kVerifyThreads) void verify_decide_kernel(const VerifyParams p) {
    __shared__ Row rows[kVerifyMaxDraft + 1];
    __shared__ uint8_t stays[kVerifyMaxDraft + 1];
    __shared__ PickLds lds;
    __shared__ double lds_d[4];
    __shared__ ExpTable table;
    const uint32_t s = blockIdx.x, lane = threadIdx.x & 63u;
    uint32_t count, all;
    const uint32_t first = rows_of(p, s, count, all);
    bool greedy;
    const double inv = inv_temperature(p, s, greedy);
    const float u_sample = p.u_sample[s];
    fill_table(table);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (uint32_t i0 = wave; i0 < count; i0 += 4 * kRowsAtOnce) {
        Part held[kRowsAtOnce][kPartsHeld];
        uint32_t id[kRowsAtOnce];
        float u[kRowsAtOnce], logit[kRowsAtOnce], q[kRowsAtOnce];
        const Part *parts[kRowsAtOnce];
        // rows behind the last are the last again
#pragma unroll
        for (int x = 0; x < kRowsAtOnce; ++x) {
            const uint32_t i = min(i0 + 4u * x, count - 1u);
            parts[x] = p.parts + (static_cast<uint64_t>(s) * (p.max_draft + 1) + i) * p.n_parts;
#pragma unroll
            for (int k = 0; k < kPartsHeld; ++k) {
                const uint32_t at = lane + 64u * k;
                held[x][k] = at < p.n_parts ? parts[x][at] : Part{0.0, -INFINITY, kNowhere};
            }
            const uint64_t r = static_cast<uint64_t>(first) + i;
            id[x] = kNowhere;
            u[x] = 0.0f;
            if (i + 1 < count) {
                id[x] = static_cast<uint32_t>(p.tokens[r + 1]);
                u[x] = p.u_accept[r];
            }
        }
#pragma unroll
        for (int x = 0; x < kRowsAtOnce; ++x) {
            const uint64_t r = static_cast<uint64_t>(first) + min(i0 + 4u * x, count - 1u);
            logit[x] = -INFINITY;
            q[x] = 1.0f;
            if (id[x] < p.n_vocab) {  // a NaN has no weight either
                logit[x] = static_cast<float>(reinterpret_cast<const T *>(p.logits + r * p.logits_nb)[id[x]]);
                if (p.probs) {
                    q[x] = load_float(p.probs + r * p.probs_nb, p.probs_type, id[x]);
                }
            }
        }
        Row row[kRowsAtOnce];
        float m[kRowsAtOnce];
#pragma unroll
        for (int x = 0; x < kRowsAtOnce; ++x) {
            m[x] = held[x][0].max;
#pragma unroll
            for (int k = 1; k < kPartsHeld; ++k) {
                m[x] = __builtin_fmaxf(m[x], held[x][k].max);
            }
            for (uint32_t at = lane + 64u * kPartsHeld; at < p.n_parts; at += 64) {
                m[x] = __builtin_fmaxf(m[x], parts[x][at].max);
            }
            row[x].max = wave_max(m[x]);
        }
#pragma unroll
        for (int x = 0; x < kRowsAtOnce; ++x) {
            const double max = row[x].max;
            uint32_t id_of_max = kNowhere;
            double sum = 0.0;
            auto add = [&](const Part &part) {
                id_of_max = part.max == row[x].max ? min(id_of_max, part.at) : id_of_max;
                sum += part.sum > 0.0 ? part.sum * weight_of(table, part.max, inv, max) : 0.0;
            };
#pragma unroll
            for (int k = 0; k < kPartsHeld; ++k) {
                add(held[x][k]);
            }
            for (uint32_t at = lane + 64u * kPartsHeld; at < p.n_parts; at += 64) {
                add(parts[x][at]);
            }
            row[x].sum = wave_sum(sum);
            row[x].at = wave_min(id_of_max);
            bool ok = false;
            if (id[x] < p.n_vocab && row[x].max > -INFINITY) {
                if (greedy || row[x].max == INFINITY) {
                    ok = id[x] == row[x].at;
                } else {
                    ok = static_cast<double>(u[x]) * static_cast<double>(q[x]) <
                         weight_of(table, logit[x], inv, max) / row[x].sum;
                }
            }
            const uint32_t i = i0 + 4u * x;
            if (lane == 0 && i < count) {
                rows[i] = row[x];
                stays[i] = ok;
            }
        }
    }
    __syncthreads();
    uint32_t accepted = 0;
    while (accepted + 1 < count && stays[accepted]) {
        ++accepted;
    }
    write_request(p, s, first, count, all, accepted);
    if (threadIdx.x == 0) {
        p.choice[s].pending = 0;
    }
    if (count == 0) {
        return;
    }
    __syncthreads();  // tokens_out[accepted] is written again below
    int32_t *token = p.tokens_out + static_cast<uint64_t>(s) * (p.max_draft + 1) + accepted;
    const Row row = rows[accepted];
    if (row.max == -INFINITY) {
        return;  // nothing to draw from: -1
    }
    if (greedy || row.max == INFINITY) {
        if (threadIdx.x == 0) {
            *token = static_cast<int32_t>(row.at);
        }
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
    const double max = row.max;
    const Part *parts = p.parts + (static_cast<uint64_t>(s) * (p.max_draft + 1) + accepted) * p.n_parts;
    const uint8_t *logits = p.logits + r * p.logits_nb;
    uint32_t without = refused ? static_cast<uint32_t>(p.tokens[r + 1]) : kNowhere;
    without = without < p.n_vocab ? without : kNowhere;
    double w[8];
    auto load_weights = [&](uint32_t v0) {
        float x[8];
        load_part<T>(logits, v0, min(p.n_vocab, v0 + kPartIds), x);
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            const double y = weight_of(table, x[i], inv, max);
            w[i] = v0 + threadIdx.x * 8u + i == without ? 0.0 : y;
        }
    };
    uint32_t cut = kNowhere;  // the draft's part, and that part's sum without it
    double cut_sum = 0.0;
    auto part_weight = [&](uint32_t i) {
        const Part part = parts[i];
        return i == cut ? cut_sum : part.sum > 0.0 ? part.sum * weight_of(table, part.max, inv, max) : 0.0;
    };
    if (without != kNowhere) {
        cut = without / kPartIds;
        load_weights(cut * kPartIds);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            cut_sum += w[i];
        }
        cut_sum = block_sum(cut_sum, lds_d);
    }
    double target = u_sample, before;
    uint32_t part = pick_part(p.n_parts, target, part_weight, lds, before);
    if (part == kNowhere && without != kNowhere) {  // the draft was all there is
        without = cut = kNowhere;
        target = u_sample;
        __syncthreads();
        part = pick_part(p.n_parts, target, part_weight, lds, before);
    }
    if (part == kNowhere) {
        return;
    }
    load_weights(part * kPartIds);
    pick_id(part * kPartIds, before, target, w, lds, token);
}

__device__ inline double rest_of(const ExpTable &table, double scale, float logit, float q, double inv,
                                 double max) {
    const double e = weight_of(table, logit, inv, max) * scale - static_cast<double>(q);
    return e > 0.0 ? e : 0.0;
}

template <typename T, typename Q>
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
    const uint32_t v0 = part * kPartIds, v1 = min(p.n_vocab, v0 + kPartIds);
    float x[8], q[8];
    load_part<T>(p.logits + r * p.logits_nb, v0, v1, x);
    load_part<Q>(p.probs + r * p.probs_nb, v0, v1, q);
    fill_table(table);
    bool greedy;
    const double inv = inv_temperature(p, s, greedy);
    const double max = c.max;
    double sum = 0.0;
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) {
        // behind the part's end logit and q are -inf
        sum += v0 + threadIdx.x * 8u + e < v1 ? rest_of(table, c.scale, x[e], q[e], inv, max) : 0.0;
    }
    sum = block_sum(sum, lds_d);
    if (threadIdx.x == 0) {
        p.rest[static_cast<uint64_t>(s) * p.n_parts + part] = sum;
    }
}

template <typename T, typename Q>
__global__ __launch_bounds__(kVerifyThreads) void verify_draw_kernel(const VerifyParams p) {
    __shared__ PickLds lds;
    __shared__ ExpTable table;
    const uint32_t s = blockIdx.x;
    const Choice c = p.choice[s];
    if (!c.pending) {
        return;
    }
    uint32_t count, all;
    const uint64_t r = static_cast<uint64_t>(rows_of(p, s, count, all)) + c.row;
    bool greedy;
    const double inv = inv_temperature(p, s, greedy);
    const float u_sample = p.u_sample[s];
    fill_table(table);
    const double *rest = p.rest + static_cast<uint64_t>(s) * p.n_parts;
    const Part *parts = p.parts + (static_cast<uint64_t>(s) * (p.max_draft + 1) + c.row) * p.n_parts;
    const double max = c.max;
    double target = u_sample, before;
    uint32_t part = pick_part(p.n_parts, target, [&](uint32_t i) { return rest[i]; }, lds, before);
    const bool left = part != kNowhere;  // else p itself
    if (!left) {
        target = u_sample;
        __syncthreads();
        part = pick_part(
            p.n_parts, target,
            [&](uint32_t i) {
                const Part x = parts[i];
                return x.sum > 0.0 ? x.sum * weight_of(table, x.max, inv, max) : 0.0;
            },
            lds, before);
    }
    if (part == kNowhere) {
        return;
    }
    const uint32_t v0 = part * kPartIds, v1 = min(p.n_vocab, v0 + kPartIds);
    float x[8], q[8];
    double w[8];
    load_part<T>(p.logits + r * p.logits_nb, v0, v1, x);
    load_part<Q>(p.probs + r * p.probs_nb, v0, v1, q);
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const double y = left ? rest_of(table, c.scale, x[i], q[i], inv, max)
                              : weight_of(table, x[i], inv, max);
        w[i] = v0 + threadIdx.x * 8u + i < v1 ? y : 0.0;  // behind the end logit and q are -inf
    }
    pick_id(v0, before, target, w, lds, p.tokens_out + static_cast<uint64_t>(s) * (p.max_draft + 1) + c.row);
}

template <typename T, typename Q>
static void launch_rest(hipStream_t stream, const VerifyParams &p) {
    verify_rest_kernel<T, Q><<<dim3(p.n_parts, p.n_seq), kVerifyThreads, 0, stream>>>(p);
    if (hipPeekAtLastError() == hipSuccess) {
        verify_draw_kernel<T, Q><<<p.n_seq, kVerifyThreads, 0, stream>>>(p);
    }
}

template <typename T>
static void launch_verify(hipStream_t stream, const VerifyParams &p) {
    const dim3 grid(p.n_parts, p.max_draft + 1, p.n_seq);
    if (static_cast<uint64_t>(p.n_parts) * (p.max_draft + 1) * p.n_seq >= kManyParts) {
        verify_parts_kernel<T, 4><<<grid, kVerifyThreads / 4, 0, stream>>>(p);
    } else {
        verify_parts_kernel<T, 1><<<grid, kVerifyThreads, 0, stream>>>(p);
    }
    if (hipPeekAtLastError() != hipSuccess) {
        return;  // parts that were not written must not be read
    }
    verify_decide_kernel<T><<<p.n_seq, kVerifyThreads, 0, stream>>>(p);
    if (!p.probs || !p.max_draft || hipPeekAtLastError() != hipSuccess) {
        return;
    }
    if (p.probs_type == KVMEM_TYPE_F32) {
        launch_rest<T, float>(stream, p);
    } else if (p.probs_type == KVMEM_TYPE_F16) {
        launch_rest<T, _Float16>(stream, p);
    } else {
        launch_rest<T, __bf16>(stream, p);
    }
}

bool load_verify_kernels() {
    return load_kernel_object(&verify_decide_kernel<float>);
}

struct VerifyPlan {
    uint32_t n_parts;
    size_t parts_bytes, rest_bytes, choice_bytes;
};

static VerifyPlan plan_verify(const kvmem_hip_verify_args *a) {
    VerifyPlan pl;
    pl.n_parts = (a->n_vocab + kPartIds - 1) / kPartIds;
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
    p.n_parts = pl.n_parts;
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
