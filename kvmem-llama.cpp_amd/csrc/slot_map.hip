// Block tables, cells and positions of the new tokens of a batch of requests,
// from their lengths, on the device (kvmem_hip_slot_map).
//
// With n[s] tokens cached and m[s] new ones, blocks of T tokens and a table of
// W entries per request:
//   q_start      exclusive prefix sums of m
//   b0 = min(ceil(n / T), W), b1 = min(ceil((n + m) / T), W)
//   first        exclusive prefix sums of b1 - b0
//   table[s][b0 + j] = free_slots[used + first[s] + j]       (b0 + j < b1)
//   cell of token i of s = table[s][p / T] * T + p % T, p = n[s] + i
// The two prefix sums are all that couples the requests.  They are small
// (a few words a request), so every workgroup computes them again in LDS
// rather than waiting for one that does: one launch, no workspace, nothing
// ordered between workgroups, and a block's slot comes from the free list
// itself, not from the table entry another workgroup writes.  Bound by latency:
// 8 requests with one token each take 4.1 us (launch, lengths, slots), 256 with up
// to 509 tokens each 8.1 us (59 workgroups, in which a thread's four tokens are four
// searches with their loads, one after another).
#include "kvmem_internal.hpp"

#include <algorithm>

namespace kvmem_hip {

constexpr uint32_t kSlotMapThreads = 256;
constexpr uint32_t kSlotMapMaxSeq = 4096;  // two prefix sums in LDS: 32 KiB
// Tokens of one workgroup (four a thread) before another is launched.
constexpr uint32_t kSlotMapTokens = 1024;

struct SlotMapParams {
    uint32_t n_seq, T, n_slots, W, max_tokens, n_free;
    const uint32_t *n_new;
    const uint32_t *kv_len;
    const int32_t *pos0;
    const uint32_t *free_slots;
    const uint32_t *free_used;
    uint32_t *table;
    uint32_t *kv_len_out;
    uint32_t *q_start;
    int32_t *positions;
    int32_t *cells;
    uint32_t *free_used_out;
    uint32_t *n_missing;
};

// Lengths come from device memory: sums that pass 32 bits stay at the top.
__device__ inline uint32_t sat_add(uint32_t a, uint32_t b) {
    const uint32_t c = a + b;
    return c < a ? 0xffffffffu : c;
}

__device__ inline uint32_t ceil_div(uint32_t a, uint32_t b) { return a / b + (a % b != 0 ? 1u : 0u); }

// The last of n + 1 nondecreasing sums (sum[0] = 0) that is at most x, x < sum[n].
__device__ inline uint32_t find_run(const uint32_t *sum, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (sum[mid] <= x) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    return lo;
}

__global__ __launch_bounds__(kSlotMapThreads) void slot_map_kernel(SlotMapParams p) {
    extern __shared__ uint32_t sums[];  // [n_seq + 1] tokens, [n_seq + 1] blocks
    __shared__ uint32_t wave_sum[3][kSlotMapThreads / 64];
    uint32_t *tok = sums;
    uint32_t *blk = sums + p.n_seq + 1;
    const uint32_t tid = threadIdx.x;
    const uint32_t lane = tid & 63u;
    const uint32_t wave = tid >> 6;

    // each thread sums a run of requests, then the runs are summed
    const uint32_t per = (p.n_seq + kSlotMapThreads - 1) / kSlotMapThreads;
    const uint32_t s0 = min(p.n_seq, tid * per);
    const uint32_t s1 = min(p.n_seq, s0 + per);
    uint32_t run[3] = {0, 0, 0};  // tokens, blocks with an entry, blocks asked for
    for (uint32_t s = s0; s < s1; ++s) {
        const uint32_t n = p.kv_len[s];
        const uint32_t m = p.n_new[s];
        const uint32_t b0 = ceil_div(n, p.T);
        const uint32_t b1 = ceil_div(sat_add(n, m), p.T);
        run[0] = sat_add(run[0], m);
        run[1] += min(b1, p.W) - min(b0, p.W);  // n_seq * W fits 32 bits
        run[2] = sat_add(run[2], b1 - b0);
    }
    uint32_t inc[3] = {run[0], run[1], run[2]};
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const uint32_t o = __shfl_up(inc[i], d, 64);
            inc[i] = lane >= d ? sat_add(inc[i], o) : inc[i];
        }
    }
    if (lane == 63u) {
        for (int i = 0; i < 3; ++i) {
            wave_sum[i][wave] = inc[i];
        }
    }
    __syncthreads();
    uint32_t base[2] = {0, 0};
    uint32_t total[3] = {0, 0, 0};
    for (uint32_t w = 0; w < kSlotMapThreads / 64; ++w) {
        for (int i = 0; i < 2; ++i) {
            base[i] = w < wave ? sat_add(base[i], wave_sum[i][w]) : base[i];
        }
        for (int i = 0; i < 3; ++i) {
            total[i] = sat_add(total[i], wave_sum[i][w]);
        }
    }
    // exclusive sum of this thread's run: the lanes before it in the wave
    uint32_t at[2];
    for (int i = 0; i < 2; ++i) {
        const uint32_t before = __shfl_up(inc[i], 1, 64);
        at[i] = sat_add(base[i], lane == 0 ? 0u : before);
    }
    const bool first_group = blockIdx.x == 0;
    for (uint32_t s = s0; s < s1; ++s) {
        const uint32_t n = p.kv_len[s];
        const uint32_t m = p.n_new[s];
        const uint32_t end = sat_add(n, m);
        tok[s] = at[0];
        blk[s] = at[1];
        if (first_group) {
            p.q_start[s] = at[0];
            p.kv_len_out[s] = end;
        }
        at[0] = sat_add(at[0], m);
        at[1] += min(ceil_div(end, p.T), p.W) - min(ceil_div(n, p.T), p.W);
    }
    if (tid == 0) {
        tok[p.n_seq] = total[0];
        blk[p.n_seq] = total[1];
    }
    const uint32_t used = min(*p.free_used, p.n_free);
    const uint32_t given = min(total[1], p.n_free - used);
    if (first_group && tid == 0) {
        p.q_start[p.n_seq] = total[0];
        *p.free_used_out = used + given;
        *p.n_missing = total[2] - given;
    }
    __syncthreads();

    const uint32_t step = gridDim.x * kSlotMapThreads;
    for (uint32_t t = blockIdx.x * kSlotMapThreads + tid; t < p.max_tokens; t += step) {
        int32_t cell = -1;
        int32_t pos = 0;
        if (t < total[0]) {
            const uint32_t s = find_run(tok, p.n_seq, t);
            const uint32_t i = t - tok[s];
            const uint32_t n = p.kv_len[s];
            const uint32_t x = n + i;  // wraps only past the table (its block is then checked first)
            const uint32_t b = x / p.T;
            const uint32_t b0 = ceil_div(n, p.T);
            pos = static_cast<int32_t>((p.pos0 ? static_cast<uint32_t>(p.pos0[s]) : n) + i);
            uint32_t slot = KVMEM_HIP_NO_SLOT;
            if (x >= n && b < p.W) {
                if (b < b0) {
                    slot = p.table[static_cast<uint64_t>(s) * p.W + b];
                } else {
                    const uint32_t f = blk[s] + (b - b0);
                    slot = f < given ? p.free_slots[used + f] : KVMEM_HIP_NO_SLOT;
                }
            }
            if (slot < p.n_slots) {
                cell = static_cast<int32_t>(slot * p.T + x % p.T);
            }
        }
        p.positions[t] = pos;
        p.cells[t] = cell;
        if (p.max_tokens - t <= step) {
            break;  // t + step may pass 32 bits
        }
    }
    for (uint32_t b = blockIdx.x * kSlotMapThreads + tid; b < total[1]; b += step) {
        const uint32_t s = find_run(blk, p.n_seq, b);
        const uint32_t e = ceil_div(p.kv_len[s], p.T) + (b - blk[s]);
        uint32_t slot = b < given ? p.free_slots[used + b] : KVMEM_HIP_NO_SLOT;
        slot = slot < p.n_slots ? slot : KVMEM_HIP_NO_SLOT;
        p.table[static_cast<uint64_t>(s) * p.W + e] = slot;
        if (total[1] - b <= step) {
            break;
        }
    }
}

bool load_slot_map_kernels() {
    return load_kernel_object(&slot_map_kernel);
}

}  // namespace kvmem_hip

using namespace kvmem_hip;

extern "C" {

int kvmem_hip_slot_map(kvmem_hip_ctx *ctx, const kvmem_hip_slot_map_args *a) {
    if (!ctx) {
        return KVMEM_HIP_ERR_INVALID;
    }
    if (!a) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "slot_map: null arguments");
    }
    if (a->n_seq == 0 || a->block_tokens == 0 || a->table_stride == 0) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "slot_map: empty geometry");
    }
    if (a->n_seq > kSlotMapMaxSeq) {
        return fail(ctx, KVMEM_HIP_ERR_UNSUPPORTED, "slot_map: at most 4096 requests");
    }
    if (!a->n_new || !a->kv_len || !a->free_used || !a->table || !a->kv_len_out || !a->q_start ||
        !a->free_used_out || !a->n_missing || (a->n_free && !a->free_slots) ||
        (a->max_tokens && (!a->positions || !a->cells))) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "slot_map: null array");
    }
    const uintptr_t all = reinterpret_cast<uintptr_t>(a->n_new) | reinterpret_cast<uintptr_t>(a->kv_len) |
                          reinterpret_cast<uintptr_t>(a->pos0) | reinterpret_cast<uintptr_t>(a->free_slots) |
                          reinterpret_cast<uintptr_t>(a->free_used) | reinterpret_cast<uintptr_t>(a->table) |
                          reinterpret_cast<uintptr_t>(a->kv_len_out) | reinterpret_cast<uintptr_t>(a->q_start) |
                          reinterpret_cast<uintptr_t>(a->positions) | reinterpret_cast<uintptr_t>(a->cells) |
                          reinterpret_cast<uintptr_t>(a->free_used_out) | reinterpret_cast<uintptr_t>(a->n_missing);
    if (all & 3u) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "slot_map: arrays must be 4-byte aligned");
    }
    if (static_cast<uint64_t>(a->n_slots) * a->block_tokens > 0x7fffffffu) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "slot_map: cells must fit 31 bits");
    }
    if (static_cast<uint64_t>(a->n_seq) * a->table_stride > 0xffffffffu) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "slot_map: table larger than 2^32 entries");
    }
    if (a->kv_len == a->kv_len_out || a->free_used == a->free_used_out) {
        return fail(ctx, KVMEM_HIP_ERR_INVALID, "slot_map: outputs must not overlap inputs");
    }
    const SlotMapParams p{a->n_seq,     a->block_tokens, a->n_slots,   a->table_stride, a->max_tokens, a->n_free,
                          a->n_new,     a->kv_len,       a->pos0,      a->free_slots,   a->free_used,  a->table,
                          a->kv_len_out, a->q_start,     a->positions, a->cells,        a->free_used_out, a->n_missing};
    (void) hipSetDevice(ctx->device);
    if (injected_fail(ctx, KVMEM_HIP_FAIL_LAUNCH, "slot_map launch")) {
        return KVMEM_HIP_ERR_RUNTIME;
    }
    const uint32_t grid = std::max(1u, std::min(1024u, a->max_tokens / kSlotMapTokens +
                                                           (a->max_tokens % kSlotMapTokens ? 1u : 0u)));
    const uint32_t lds = 2u * (a->n_seq + 1u) * sizeof(uint32_t);
    slot_map_kernel<<<grid, kSlotMapThreads, lds, ctx->stream>>>(p);
    return hip_ok(ctx, hipGetLastError(), "slot_map launch") ? KVMEM_HIP_OK : KVMEM_HIP_ERR_RUNTIME;
}

}  // extern "C"
