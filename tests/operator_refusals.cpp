// Refusals of kvmem_hip_slot_map, kvmem_hip_qkv_rows and kvmem_hip_attention:
// every call here must be turned away by the host checks, before any HIP call,
// so the program runs without a GPU.  Linked with libkvmem_hip.so; the context
// is a bare struct (no stream, no device).
#include <cstdio>
#include <cstring>
#include <functional>
#include <string>

#include "kvmem_internal.hpp"

static int bad = 0;
static kvmem_hip_ctx ctx;

static void expect(const char *what, int want, int got) {
    const std::string said = kvmem_hip_last_error(&ctx);
    if (got != want || said.empty()) {
        std::printf("%s: status %d, expected %d (%s)\n", what, got, want, said.c_str());
        ++bad;
    }
    ctx.last_error.clear();
}

// addresses that are checked, never followed
static void *const A = reinterpret_cast<void *>(uintptr_t{0x10000});
static void *const OFF4 = reinterpret_cast<void *>(uintptr_t{0x10004});
static void *const OFF1 = reinterpret_cast<void *>(uintptr_t{0x10001});
static void *layers[1] = {A};
static void *no_layer[1] = {nullptr};
static void *off_layer[1] = {OFF4};
static float theta[256];

static void slot_map() {
    using Args = kvmem_hip_slot_map_args;
    auto *u = static_cast<uint32_t *>(A);
    auto *i = static_cast<int32_t *>(A);
    Args ok{};
    ok.n_seq = 2, ok.block_tokens = 128, ok.n_slots = 8, ok.table_stride = 4, ok.max_tokens = 2, ok.n_free = 1;
    ok.n_new = ok.kv_len = ok.free_slots = ok.free_used = u;
    ok.kv_len_out = ok.table = ok.q_start = ok.free_used_out = ok.n_missing = u + 64;
    ok.positions = ok.cells = i;
    auto call = [&](const char *what, int want, const std::function<void(Args &)> &f) {
        Args a = ok;
        f(a);
        expect(what, want, kvmem_hip_slot_map(&ctx, &a));
    };
    const int inv = KVMEM_HIP_ERR_INVALID;
    expect("null args", inv, kvmem_hip_slot_map(&ctx, nullptr));
    call("no requests", inv, [](Args &a) { a.n_seq = 0; });
    call("no block tokens", inv, [](Args &a) { a.block_tokens = 0; });
    call("no table", inv, [](Args &a) { a.table_stride = 0; });
    call("too many requests", KVMEM_HIP_ERR_UNSUPPORTED, [](Args &a) { a.n_seq = 4097; });
    call("null n_new", inv, [](Args &a) { a.n_new = nullptr; });
    call("null kv_len", inv, [](Args &a) { a.kv_len = nullptr; });
    call("null free_used", inv, [](Args &a) { a.free_used = nullptr; });
    call("null free_slots", inv, [](Args &a) { a.free_slots = nullptr; });
    call("null table", inv, [](Args &a) { a.table = nullptr; });
    call("null kv_len_out", inv, [](Args &a) { a.kv_len_out = nullptr; });
    call("null q_start", inv, [](Args &a) { a.q_start = nullptr; });
    call("null positions", inv, [](Args &a) { a.positions = nullptr; });
    call("null cells", inv, [](Args &a) { a.cells = nullptr; });
    call("null free_used_out", inv, [](Args &a) { a.free_used_out = nullptr; });
    call("null n_missing", inv, [](Args &a) { a.n_missing = nullptr; });
    call("odd address", inv, [](Args &a) { a.cells = static_cast<int32_t *>(OFF1); });
    call("cells past 31 bits", inv, [](Args &a) { a.n_slots = 1u << 24; });
    call("table past 32 bits", inv, [](Args &a) { a.n_seq = 4096, a.table_stride = 1u << 20; });
    call("lengths in place", inv, [](Args &a) { a.kv_len_out = const_cast<uint32_t *>(a.kv_len); });
    call("count in place", inv, [](Args &a) { a.free_used_out = const_cast<uint32_t *>(a.free_used); });
}

static void qkv_rows() {
    using Args = kvmem_hip_qkv_args;
    kvmem_hip_transform xf{128, 64, theta, 128, 64, nullptr};
    kvmem_hip_pool pool{1, 8, 128, 512, 512, KVMEM_TYPE_Q4_0, KVMEM_TYPE_Q8_0, layers, layers, &xf};
    Args ok{};
    ok.q = ok.k = ok.v = A;
    ok.type = ok.out_type = KVMEM_TYPE_F16;
    ok.n_tokens = 3, ok.n_head = 8, ok.n_head_kv = 4, ok.head_dim = 128;
    ok.q_nb1 = ok.k_nb1 = ok.v_nb1 = 256, ok.q_nb2 = 2048, ok.k_nb2 = ok.v_nb2 = 1024;
    ok.positions = ok.cells = static_cast<int32_t *>(A);
    ok.q_out = A;
    auto call = [&](const char *what, int want, const std::function<void(Args &, kvmem_hip_pool &)> &f,
                    uint32_t layer = 0) {
        Args a = ok;
        kvmem_hip_pool p = pool;
        f(a, p);
        expect(what, want, kvmem_hip_qkv_rows(&ctx, &p, layer, &a));
    };
    const int inv = KVMEM_HIP_ERR_INVALID;
    const int uns = KVMEM_HIP_ERR_UNSUPPORTED;
    expect("rows: null args", inv, kvmem_hip_qkv_rows(&ctx, &pool, 0, nullptr));
    expect("rows: no pool for v", inv, kvmem_hip_qkv_rows(&ctx, nullptr, 0, &ok));
    call("rows: quantized input", uns, [](Args &a, kvmem_hip_pool &) { a.type = KVMEM_TYPE_Q8_0; });
    call("rows: quantized output", uns, [](Args &a, kvmem_hip_pool &) { a.out_type = KVMEM_TYPE_Q8_0; });
    for (uint32_t d : {0u, 32u, 96u, 1024u}) {
        call("rows: head_dim", uns, [d](Args &a, kvmem_hip_pool &) { a.head_dim = d; });
    }
    call("rows: no heads", inv, [](Args &a, kvmem_hip_pool &) { a.n_head = 0; });
    call("rows: no KV heads", inv, [](Args &a, kvmem_hip_pool &) { a.n_head_kv = 0; });
    call("rows: too many heads", inv, [](Args &a, kvmem_hip_pool &) { a.n_head = 4097; });
    call("rows: too many tokens", inv, [](Args &a, kvmem_hip_pool &) { a.n_tokens = (1u << 26) + 1; });
    call("rows: nothing given", inv, [](Args &a, kvmem_hip_pool &) { a.q = a.k = a.v = nullptr; });
    call("rows: q without output", inv, [](Args &a, kvmem_hip_pool &) { a.q_out = nullptr; });
    call("rows: transform's head_dim", inv, [&](Args &, kvmem_hip_pool &p) {
        static kvmem_hip_transform x;
        x = xf, x.head_dim = 64, p.xf = &x;
    });
    for (uint32_t r : {8u, 72u, 144u}) {
        call("rows: n_rot", inv, [&](Args &a, kvmem_hip_pool &) {
            static kvmem_hip_transform x;
            x = xf, x.n_rot = r, a.xf = &x;
        });
    }
    call("rows: no theta", inv, [&](Args &a, kvmem_hip_pool &) {
        static kvmem_hip_transform x;
        x = xf, x.theta = nullptr, a.xf = &x;
    });
    call("rows: no positions", inv, [](Args &a, kvmem_hip_pool &) { a.positions = nullptr; });
    for (uint32_t w : {16u, 96u, 256u}) {
        call("rows: hadamard_k", inv, [&](Args &a, kvmem_hip_pool &) {
            static kvmem_hip_transform x;
            x = xf, x.hadamard_k = w, a.xf = &x;
        });
    }
    call("rows: odd stride", inv, [](Args &a, kvmem_hip_pool &) { a.k_nb2 = 1023; });
    call("rows: odd address", inv, [](Args &a, kvmem_hip_pool &) { a.v = OFF1; });
    call("rows: output address", inv, [](Args &a, kvmem_hip_pool &) { a.q_out = OFF4; });
    call("rows: weight address", inv, [](Args &a, kvmem_hip_pool &) { a.k_weight = static_cast<float *>(OFF4); });
    call("rows: layer", inv, [](Args &, kvmem_hip_pool &) {}, 1);
    call("rows: no cells", inv, [](Args &a, kvmem_hip_pool &) { a.cells = nullptr; });
    call("rows: row width", inv, [](Args &, kvmem_hip_pool &p) { p.n_embd_k = 256; });
    call("rows: value width", inv, [](Args &, kvmem_hip_pool &p) { p.n_embd_v = 1024; });
    call("rows: cache type", uns, [](Args &, kvmem_hip_pool &p) { p.type_v = KVMEM_TYPE_BF16; });
    call("rows: no value tensors", inv, [](Args &, kvmem_hip_pool &p) { p.v_layers = nullptr; });
    call("rows: null layer", inv, [](Args &, kvmem_hip_pool &p) { p.k_layers = no_layer; });
    call("rows: layer address", inv, [](Args &, kvmem_hip_pool &p) { p.k_layers = off_layer; });
    call("rows: pool past 31 bits", inv, [](Args &, kvmem_hip_pool &p) { p.n_slots = 1u << 24; });
}

static void attention() {
    using Args = kvmem_hip_attn_args;
    kvmem_hip_transform xf{128, 0, nullptr, 128, 64, nullptr};
    kvmem_hip_pool pool{1, 8, 128, 512, 512, KVMEM_TYPE_Q4_0, KVMEM_TYPE_Q8_0, layers, layers, &xf};
    Args ok{};
    ok.q = A, ok.q_type = KVMEM_TYPE_BF16, ok.out_type = KVMEM_TYPE_F32, ok.q_nb1 = 256, ok.q_nb2 = 2048, ok.out = A;
    ok.n_tokens = 4, ok.n_seq = 2, ok.max_q = 2, ok.max_kv = 1000, ok.n_head = 8, ok.n_head_kv = 4, ok.head_dim = 128;
    ok.table_stride = 8;
    ok.q_start = ok.kv_len = ok.table = static_cast<uint32_t *>(A);
    auto call = [&](const char *what, int want, const std::function<void(Args &, kvmem_hip_pool &)> &f,
                    uint32_t layer = 0) {
        Args a = ok;
        kvmem_hip_pool p = pool;
        f(a, p);
        expect(what, want, kvmem_hip_attention(&ctx, &p, layer, &a));
    };
    const int inv = KVMEM_HIP_ERR_INVALID;
    const int uns = KVMEM_HIP_ERR_UNSUPPORTED;
    expect("null args", inv, kvmem_hip_attention(&ctx, &pool, 0, nullptr));
    expect("null pool", inv, kvmem_hip_attention(&ctx, nullptr, 0, &ok));
    call("no q", inv, [](Args &a, kvmem_hip_pool &) { a.q = nullptr; });
    call("no out", inv, [](Args &a, kvmem_hip_pool &) { a.out = nullptr; });
    call("no kv_len", inv, [](Args &a, kvmem_hip_pool &) { a.kv_len = nullptr; });
    call("no table", inv, [](Args &a, kvmem_hip_pool &) { a.table = nullptr; });
    call("empty table", inv, [](Args &a, kvmem_hip_pool &) { a.table_stride = 0; });
    call("no heads", inv, [](Args &a, kvmem_hip_pool &) { a.n_head = 0; });
    call("no KV heads", inv, [](Args &a, kvmem_hip_pool &) { a.n_head_kv = 0; });
    call("uneven heads", inv, [](Args &a, kvmem_hip_pool &) { a.n_head = 9; });
    call("too many heads", inv, [](Args &a, kvmem_hip_pool &) { a.n_head = 8192; });
    call("tokens for requests", inv, [](Args &a, kvmem_hip_pool &) { a.q_start = nullptr, a.n_tokens = 1; });
    call("q address", inv, [](Args &a, kvmem_hip_pool &) { a.q = OFF4; });
    call("q head stride", inv, [](Args &a, kvmem_hip_pool &) { a.q_nb1 = 258; });
    call("q token stride", inv, [](Args &a, kvmem_hip_pool &) { a.q_nb2 = 2056; });
    call("out address", inv, [](Args &a, kvmem_hip_pool &) { a.out = OFF4; });
    call("lse address", inv, [](Args &a, kvmem_hip_pool &) { a.lse = static_cast<float *>(OFF1); });
    call("too many requests", inv, [](Args &a, kvmem_hip_pool &) { a.n_seq = 65536, a.n_tokens = 65536; });
    call("too many tokens", inv, [](Args &a, kvmem_hip_pool &) { a.n_tokens = (1u << 20) + 1; });
    call("too many keys", inv, [](Args &a, kvmem_hip_pool &) { a.max_kv = 0x80000000u; });
    call("negative scale", inv, [](Args &a, kvmem_hip_pool &) { a.scale = -1.0f; });
    call("NaN scale", inv, [](Args &a, kvmem_hip_pool &) { a.scale = __builtin_nanf(""); });
    call("infinite scale", inv, [](Args &a, kvmem_hip_pool &) { a.scale = __builtin_inff(); });
    call("pool past 31 bits", inv, [](Args &, kvmem_hip_pool &p) { p.n_slots = 1u << 24; });
    call("no block tokens", inv, [](Args &, kvmem_hip_pool &p) { p.block_tokens = 0; });
    call("row width", inv, [](Args &, kvmem_hip_pool &p) { p.n_embd_k = 1024; });
    call("value width", inv, [](Args &, kvmem_hip_pool &p) { p.n_embd_v = 256; });
    for (uint32_t w : {32u, 96u, 256u}) {
        call("hadamard_v", inv, [&](Args &, kvmem_hip_pool &p) {
            static kvmem_hip_transform x;
            x = xf, x.hadamard_v = w, p.xf = &x;
        });
    }
    call("transform's head_dim", inv, [&](Args &, kvmem_hip_pool &p) {
        static kvmem_hip_transform x;
        x = xf, x.head_dim = 256, p.xf = &x;
    });
    for (uint32_t d : {32u, 96u, 512u}) {
        call("head_dim", uns, [d](Args &a, kvmem_hip_pool &p) {
            a.head_dim = d, p.n_embd_k = p.n_embd_v = 4 * d, p.xf = nullptr;
        });
    }
    call("f32 queries", uns, [](Args &a, kvmem_hip_pool &) { a.q_type = KVMEM_TYPE_F32; });
    call("quantized output", uns, [](Args &a, kvmem_hip_pool &) { a.out_type = KVMEM_TYPE_Q8_0; });
    call("key type", uns, [](Args &, kvmem_hip_pool &p) { p.type_k = KVMEM_TYPE_BF16; });
    call("value type", uns, [](Args &, kvmem_hip_pool &p) { p.type_v = 3; });
    call("layer", inv, [](Args &, kvmem_hip_pool &) {}, 1);
    call("null layer", inv, [](Args &, kvmem_hip_pool &p) { p.v_layers = no_layer; });
    call("layer address", inv, [](Args &, kvmem_hip_pool &p) { p.k_layers = off_layer; });
    call("no value tensors", inv, [](Args &, kvmem_hip_pool &p) { p.v_layers = nullptr; });
    call("pool without slots", inv, [](Args &, kvmem_hip_pool &p) { p.n_slots = 0; });
    call("too large a launch", inv, [](Args &a, kvmem_hip_pool &) {
        a.n_seq = 65535, a.n_tokens = a.max_q = 1u << 20;
    });
    // 8000 keys are split: tokens x heads x parts x (128 floats and two)
    auto split = [](Args &a, kvmem_hip_pool &p) {
        a.n_seq = 1, a.max_kv = 8000, a.table_stride = 64, p.n_slots = 64;
    };
    Args wide = ok;
    kvmem_hip_pool slots = pool;
    split(wide, slots);
    const size_t need = kvmem_hip_attention_workspace(&slots, &wide);
    if (need == 0 || need % (wide.n_tokens * 8 * (128 + 2) * sizeof(float)) != 0) {
        std::printf("workspace of a split call: %zu bytes\n", need);
        ++bad;
    }
    call("workspace too small", inv, [&](Args &a, kvmem_hip_pool &p) {
        split(a, p), a.workspace = A, a.workspace_bytes = need - 1;
    });
    call("workspace address", inv, [&](Args &a, kvmem_hip_pool &p) {
        split(a, p), a.workspace = OFF4, a.workspace_bytes = need;
    });
    if (kvmem_hip_attention_workspace(nullptr, &ok) != 0 || kvmem_hip_attention_workspace(&pool, nullptr) != 0) {
        std::printf("workspace of a refused call is not 0\n");
        ++bad;
    }
    if (kvmem_hip_slot_map(nullptr, nullptr) != inv || kvmem_hip_qkv_rows(nullptr, &pool, 0, nullptr) != inv ||
        kvmem_hip_attention(nullptr, &pool, 0, &ok) != inv) {
        std::printf("a null context is not refused\n");
        ++bad;
    }
}

int main() {
    slot_map();
    qkv_rows();
    attention();
    std::printf(bad ? "%d refusals differ\n" : "all refused\n", bad);
    return bad ? 1 : 0;
}
