// Refusals of kvmem_hip_conv_rows, kvmem_hip_linear_attention and
// kvmem_hip_verify_draft: every call here must be turned away by the host checks,
// before any HIP call, so the program runs without a GPU.  Linked with
// libkvmem_hip.so; the context is a bare struct (no stream, no device).
#include <cmath>
#include <cstdio>
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

static void size(const char *what, size_t want, size_t got) {
    if (want != got) {
        std::printf("%s: %zu bytes, expected %zu\n", what, got, want);
        ++bad;
    }
}

// addresses that are checked, never followed
static void *at(uintptr_t a) { return reinterpret_cast<void *>(a); }
static void *const A = at(0x10000), *const B = at(0x20000), *const C = at(0x30000);
static void *const OFF4 = at(0x10004), *const OFF2 = at(0x10002), *const OFF1 = at(0x10001);
static constexpr int inv = KVMEM_HIP_ERR_INVALID, uns = KVMEM_HIP_ERR_UNSUPPORTED;

static void conv() {
    using Args = kvmem_hip_conv_args;
    Args ok{};
    ok.x = A, ok.type = KVMEM_TYPE_BF16, ok.x_nb = 512, ok.n_tokens = 4, ok.n_seq = 2, ok.max_q = 2;
    ok.n_channels = 256, ok.width = 4, ok.n_slots = 2, ok.norm_channels = 128, ok.norm_dim = 64, ok.eps = 1e-6f;
    ok.weight = static_cast<float *>(A), ok.state = B, ok.state_out = B, ok.out = C;
    auto call = [&](const char *what, int want, const std::function<void(Args &)> &f) {
        Args a = ok;
        f(a);
        expect(what, want, kvmem_hip_conv_rows(&ctx, &a));
    };
    expect("conv: null args", inv, kvmem_hip_conv_rows(&ctx, nullptr));
    call("conv: type", uns, [](Args &a) { a.type = KVMEM_TYPE_Q8_0; });
    call("conv: width 1", uns, [](Args &a) { a.width = 1; });
    call("conv: width 9", uns, [](Args &a) { a.width = 9; });
    call("conv: no channels", inv, [](Args &a) { a.n_channels = 0; });
    call("conv: too many channels", inv, [](Args &a) { a.n_channels = (1u << 24) + 1; });
    call("conv: norm run", uns, [](Args &a) { a.norm_dim = 48; });
    call("conv: norm run too short", uns, [](Args &a) { a.norm_dim = 16; });
    call("conv: norm run too long", uns, [](Args &a) { a.norm_dim = 1024; });
    call("conv: half a run", inv, [](Args &a) { a.norm_channels = 96; });
    call("conv: runs past the channels", inv, [](Args &a) { a.norm_channels = 320; });
    call("conv: negative eps", inv, [](Args &a) { a.eps = -1.0f; });
    call("conv: NaN eps", inv, [](Args &a) { a.eps = std::nanf(""); });
    call("conv: too many requests", uns, [](Args &a) { a.n_seq = 65536; });
    call("conv: too many tokens", inv, [](Args &a) { a.n_tokens = (1u << 26) + 1; });
    call("conv: no destination", inv, [](Args &a) { a.out = nullptr, a.state_out = nullptr; });
    call("conv: null rows", inv, [](Args &a) { a.x = nullptr; });
    call("conv: null weights", inv, [](Args &a) { a.weight = nullptr; });
    call("conv: odd row address", inv, [](Args &a) { a.x = OFF1; });
    call("conv: odd stride", inv, [](Args &a) { a.x_nb = 511; });
    call("conv: odd out", inv, [](Args &a) { a.out = OFF1; });
    call("conv: weights off their size", inv, [](Args &a) { a.weight = static_cast<float *>(OFF2); });
    call("conv: slots off their size", inv, [](Args &a) { a.slots = static_cast<uint32_t *>(OFF2); });
    call("conv: out in place", inv, [](Args &a) { a.out = const_cast<void *>(a.x); });
    call("conv: out over the state", inv, [](Args &a) { a.out = a.state_out; });
    uint32_t starts = 0;
    call("conv: launch", inv, [&](Args &a) {
        a.q_start = &starts, a.n_seq = 65535, a.max_q = a.n_tokens = 1u << 26, a.n_channels = 1u << 24;
    });
}

static void linear() {
    using Args = kvmem_hip_linear_args;
    Args ok{};
    ok.q = ok.k = ok.v = A, ok.type = ok.out_type = KVMEM_TYPE_BF16;
    ok.q_nb1 = ok.k_nb1 = ok.v_nb1 = 256, ok.q_nb2 = ok.k_nb2 = ok.v_nb2 = 4096;
    ok.n_tokens = 100, ok.n_seq = 1, ok.max_q = 100, ok.n_head_k = 2, ok.n_head = 4, ok.head_dim_k = ok.head_dim_v = 128;
    ok.n_slots = 1, ok.state = static_cast<float *>(B), ok.state_out = static_cast<float *>(B), ok.out = C;
    uint32_t starts[2] = {};
    ok.q_start = starts;
    auto call = [&](const char *what, int want, const std::function<void(Args &)> &f) {
        Args a = ok;
        f(a);
        expect(what, want, kvmem_hip_linear_attention(&ctx, &a));
        size(what, 0, kvmem_hip_linear_attention_workspace(&a));
    };
    expect("linear: null args", inv, kvmem_hip_linear_attention(&ctx, nullptr));
    size("linear: null args", 0, kvmem_hip_linear_attention_workspace(nullptr));
    Args none = ok;
    none.n_seq = 0, none.beta = nullptr, none.max_q = none.n_tokens = 1u << 20;
    size("linear: no requests", 0, kvmem_hip_linear_attention_workspace(&none));
    call("linear: type", uns, [](Args &a) { a.type = KVMEM_TYPE_Q4_0; });
    call("linear: out type", uns, [](Args &a) { a.out_type = KVMEM_TYPE_Q4_0; });
    for (uint32_t d : {0u, 32u, 96u, 512u}) {
        call("linear: key size", uns, [d](Args &a) { a.head_dim_k = d; });
    }
    for (uint32_t d : {0u, 16u, 100u, 544u}) {
        call("linear: value size", uns, [d](Args &a) { a.head_dim_v = d; });
    }
    call("linear: no heads", inv, [](Args &a) { a.n_head = 0; });
    call("linear: no key heads", inv, [](Args &a) { a.n_head_k = 0; });
    call("linear: heads not a multiple", inv, [](Args &a) { a.n_head = 3; });
    call("linear: too many heads", inv, [](Args &a) { a.n_head = 4098; });
    call("linear: too many requests", uns, [](Args &a) { a.n_seq = 65536; });
    call("linear: too many tokens", inv, [](Args &a) { a.n_tokens = (1u << 26) + 1; });
    call("linear: no destination", inv, [](Args &a) { a.out = nullptr, a.state_out = nullptr; });
    call("linear: null keys", inv, [](Args &a) { a.k = nullptr; });
    call("linear: null values", inv, [](Args &a) { a.v = nullptr; });
    call("linear: null queries", inv, [](Args &a) { a.q = nullptr; });
    call("linear: keys off 16 bytes", inv, [](Args &a) { a.k = OFF4; });
    call("linear: stride off 16 bytes", inv, [](Args &a) { a.v_nb2 = 4104; });
    call("linear: state off 16 bytes", inv, [](Args &a) { a.state = static_cast<float *>(OFF4); });
    call("linear: out off 16 bytes", inv, [](Args &a) { a.out = OFF4; });
    call("linear: gates off their size", inv, [](Args &a) { a.beta = static_cast<float *>(OFF2); });
    call("linear: gates' stride", inv, [](Args &a) { a.decay_nb = 6; });
    call("linear: out in place", inv, [](Args &a) { a.out = const_cast<void *>(a.v); });
    call("linear: out over the state", inv, [](Args &a) { a.out = a.state_out; });
    call("linear: negative scale", inv, [](Args &a) { a.scale = -1.0f; });
    call("linear: infinite scale", inv, [](Args &a) { a.scale = INFINITY; });
    call("linear: NaN scale", inv, [](Args &a) { a.scale = std::nanf(""); });
    call("linear: launch", inv, [](Args &a) { a.n_seq = 65535, a.n_head = 4096, a.max_q = 1; });
    call("linear: launch of chunks", inv, [](Args &a) { a.n_seq = 4096, a.max_q = a.n_tokens = 1u << 26; });
    const size_t need = kvmem_hip_linear_attention_workspace(&ok);
    if (need == 0) {
        std::printf("a prompt needs no workspace\n");
        ++bad;
    }
    Args a = ok;
    a.workspace = A, a.workspace_bytes = need - 1;
    expect("linear: workspace too small", inv, kvmem_hip_linear_attention(&ctx, &a));
    a.workspace = OFF4, a.workspace_bytes = need;
    expect("linear: workspace address", inv, kvmem_hip_linear_attention(&ctx, &a));
}

static void verify() {
    using Args = kvmem_hip_verify_args;
    Args ok{};
    auto *f = static_cast<float *>(A);
    auto *u = static_cast<uint32_t *>(B);
    ok.logits = A, ok.type = KVMEM_TYPE_F32, ok.logits_nb = 4000, ok.n_vocab = 1000, ok.n_rows = 8, ok.n_seq = 2, ok.max_draft = 3;
    ok.tokens = static_cast<int32_t *>(A), ok.u_accept = ok.u_sample = f;
    ok.tokens_out = static_cast<int32_t *>(B), ok.n_accepted = u, ok.n_keep = u + 16;
    auto call = [&](const char *what, int want, const std::function<void(Args &)> &g) {
        Args a = ok;
        g(a);
        expect(what, want, kvmem_hip_verify_draft(&ctx, &a));
    };
    expect("verify: null args", inv, kvmem_hip_verify_draft(&ctx, nullptr));
    size("verify: null args", 0, kvmem_hip_verify_draft_workspace(nullptr));
    call("verify: type", uns, [](Args &a) { a.type = KVMEM_TYPE_Q8_0; });
    call("verify: probabilities' type", uns, [](Args &a) { a.probs = A, a.probs_type = KVMEM_TYPE_Q8_0; });
    call("verify: too many requests", uns, [](Args &a) { a.n_seq = 65536; });
    call("verify: too many drafts", uns, [](Args &a) { a.max_draft = 128; });
    call("verify: too many ids", uns, [](Args &a) { a.n_vocab = (1u << 24) + 1; });
    call("verify: no ids", inv, [](Args &a) { a.n_vocab = 0; });
    call("verify: null logits", inv, [](Args &a) { a.logits = nullptr; });
    call("verify: null tokens", inv, [](Args &a) { a.tokens = nullptr; });
    call("verify: null u_accept", inv, [](Args &a) { a.u_accept = nullptr; });
    call("verify: null u_sample", inv, [](Args &a) { a.u_sample = nullptr; });
    call("verify: null tokens_out", inv, [](Args &a) { a.tokens_out = nullptr; });
    call("verify: null n_accepted", inv, [](Args &a) { a.n_accepted = nullptr; });
    call("verify: lengths without an output", inv, [&](Args &a) { a.kv_len = u; });
    call("verify: an output without lengths", inv, [&](Args &a) { a.kv_len_out = u; });
    call("verify: logits off their size", inv, [](Args &a) { a.logits = OFF2; });
    call("verify: rows off their size", inv, [](Args &a) { a.logits_nb = 4002; });
    call("verify: probabilities off their size", inv, [](Args &a) { a.probs = OFF1, a.probs_type = KVMEM_TYPE_F16; });
    call("verify: tokens off their size", inv, [](Args &a) { a.tokens = static_cast<int32_t *>(OFF2); });
    call("verify: tokens in place", inv, [](Args &a) { a.tokens_out = const_cast<int32_t *>(a.tokens); });
    call("verify: launch", inv, [](Args &a) { a.n_seq = 65535, a.max_draft = 127, a.n_vocab = 1u << 24; });
    const size_t need = kvmem_hip_verify_draft_workspace(&ok);
    Args a = ok;
    a.workspace = A, a.workspace_bytes = need - 1;
    expect("verify: workspace too small", inv, kvmem_hip_verify_draft(&ctx, &a));
    a.workspace = OFF4, a.workspace_bytes = need;
    expect("verify: workspace address", inv, kvmem_hip_verify_draft(&ctx, &a));
}

int main() {
    conv();
    linear();
    verify();
    kvmem_hip_conv_args c{};
    kvmem_hip_linear_args l{};
    kvmem_hip_verify_args v{};
    if (kvmem_hip_conv_rows(nullptr, &c) != inv || kvmem_hip_linear_attention(nullptr, &l) != inv ||
        kvmem_hip_verify_draft(nullptr, &v) != inv) {
        std::printf("a null context is not refused\n");
        ++bad;
    }
    std::printf(bad ? "%d refusals differ\n" : "all refused\n", bad);
    return bad ? 1 : 0;
}
