// Attention and the token log probabilities through the C++ shim: the pointer and Tensor overloads against the C ABI, bit for bit,
// and the types and sizes they refuse.  With the argument "host" only the refusals, which need no GPU.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "llmq_kernels.hpp"

static int failures = 0;
static void expect(bool ok, const char* what) {
    std::printf("%s %s\n", ok ? "ok  " : "FAIL", what);
    failures += !ok;
}
template <class F> static void refused(F f, const char* what) {
    bool threw = false;
    try { f(); } catch (const std::invalid_argument&) { threw = true; }
    expect(threw, what);
}
static Tensor tensor(ETensorDType type, void* data, std::vector<long> sizes) {
    Tensor t;
    t.DType = type, t.Data = static_cast<std::byte*>(data), t.Rank = (int)sizes.size(), t.Device = 0;
    for (std::size_t i = 0; i < sizes.size(); ++i) t.Sizes[i] = sizes[i];
    return t;
}
static void* device(std::size_t bytes, const void* from = nullptr) {
    void* p = nullptr;
    if (hipMalloc(&p, bytes + 256) != hipSuccess) std::exit(3);
    if (from && hipMemcpy(p, from, bytes, hipMemcpyHostToDevice) != hipSuccess) std::exit(3);
    return p;
}
static bool equal(const void* a, const void* b, std::size_t bytes) {
    std::vector<char> x(bytes), y(bytes);
    if (hipMemcpy(x.data(), a, bytes, hipMemcpyDeviceToHost) != hipSuccess || hipMemcpy(y.data(), b, bytes, hipMemcpyDeviceToHost) != hipSuccess)
        std::exit(3);
    return std::memcmp(x.data(), y.data(), bytes) == 0;
}

static void refusals() {
    alignas(16) static char buf[4096];
    using T = ETensorDType;
    Tensor bf = tensor(T::BF16, buf, {1, 8, 256}), out = tensor(T::BF16, buf + 1024, {1, 8, 128}), f32 = tensor(T::FP32, buf, {2, 8}), none;
    Tensor ints = tensor(T::INT32, buf, {1, 8}), bytes = tensor(T::BYTE, buf, {64});
    refused([&] { attention_forward(out, bf, bf, none, nullptr, 0.1f, 1, 8, 2, 1, 64, nullptr); }, "attention_forward: lse in bf16");
    refused([&] { attention_forward(out, f32, f32, none, nullptr, 0.1f, 1, 8, 2, 1, 64, nullptr); }, "attention_forward: qkv in fp32");
    refused([&] { attention_forward(out, f32, bf, f32, nullptr, 0.1f, 1, 8, 2, 1, 64, nullptr); }, "attention_forward: first_key in fp32");
    refused([&] { attention_forward(out, f32, bf, none, nullptr, 0.1f, 1, 8, 2, 1, 60, nullptr); }, "attention_forward: head_dim 60");
    refused([&] { attention_backward(f32, out, out, f32, bf, none, bytes, 0.1f, 1, 8, 2, 1, 64, nullptr); }, "attention_backward: dqkv in fp32");
    refused([&] { attention_backward(bf, out, out, f32, out, none, bytes, 0.1f, 1, 8, 2, 1, 64, nullptr); }, "attention_backward: little scratch");
    refused([&] { token_logprobs(f32, f32, f32, none, none, ints, ints, none, 2, 8, 8, 0, nullptr); }, "token_logprobs: logits in int32");
    refused([&] { token_logprobs(f32, f32, f32, none, none, bf, ints, none, 2, 9, 8, 0, nullptr); }, "token_logprobs: V > P");
    refused([&] { token_logprobs(f32, f32, f32, none, none, bf, ints, none, 2, 8, 8, 3, nullptr); }, "token_logprobs: no place for the top tokens");
    refused([&] { token_logprobs_backward(bf, f32, none, f32, ints, f32, none, nullptr, 2, 8, 8, nullptr); }, "token_logprobs_backward: two types");
    refused([&] { token_logprobs_backward(bf, f32, f32, bf, ints, f32, none, nullptr, 2, 8, 8, nullptr); }, "token_logprobs_backward: no entropy");
}

static void calls() {
    using T = ETensorDType;
    const int B = 2, S = 150, Nq = 4, Nkv = 2, HD = 64, C = (Nq + 2 * Nkv) * HD, O = Nq * HD;
    const std::size_t nq = (std::size_t)B * S * C, no = (std::size_t)B * S * O, nl = (std::size_t)B * Nq * S;
    std::vector<std::uint16_t> host(nq);
    std::uint32_t r = 12345;
    for (auto& v : host) r = r * 1664525u + 1013904223u, v = (std::uint16_t)(((r >> 16) & 0x80FFu) | 0x3F00u);   // +-0.5 .. 2
    std::vector<std::int32_t> first((std::size_t)B * S);
    for (int i = 0; i < B * S; ++i) first[i] = i % S / 40 * 40;
    auto* qkv = static_cast<__hip_bfloat16*>(device(nq * 2, host.data()));
    auto* dout = static_cast<__hip_bfloat16*>(device(no * 2, host.data()));
    auto* fk = static_cast<std::int32_t*>(device(first.size() * 4, first.data()));
    __hip_bfloat16 *out[3], *dqkv[3];
    float *lse[3], *am[3];
    const std::size_t need = get_attention_backward_scratch_size(B, S, Nq, Nkv, HD);
    auto* scratch = static_cast<std::byte*>(device(need));
    for (int i = 0; i < 3; ++i) {
        out[i] = static_cast<__hip_bfloat16*>(device(no * 2)), dqkv[i] = static_cast<__hip_bfloat16*>(device(nq * 2));
        lse[i] = static_cast<float*>(device(nl * 4)), am[i] = static_cast<float*>(device(4));
        if (i == 0) {
            llmq_detail::check(llmq_attention_forward_bf16(llmq_detail::u16(out[0]), lse[0], llmq_detail::u16(qkv), fk, am[0], 0.125f, B, S, Nq, Nkv, HD, nullptr));
            llmq_detail::check(llmq_attention_backward_bf16(llmq_detail::u16(dqkv[0]), llmq_detail::u16(dout), llmq_detail::u16(out[0]), lse[0],
                                                            llmq_detail::u16(qkv), fk, scratch, need, 0.125f, B, S, Nq, Nkv, HD, nullptr));
        } else if (i == 1) {
            attention_forward(out[1], lse[1], qkv, fk, am[1], 0.125f, B, S, Nq, Nkv, HD, nullptr);
            attention_backward(dqkv[1], dout, out[1], lse[1], qkv, fk, scratch, need, 0.125f, B, S, Nq, Nkv, HD, nullptr);
        } else {
            Tensor o = tensor(T::BF16, out[2], {B, S, O}), l = tensor(T::FP32, lse[2], {B, Nq, S}), x = tensor(T::BF16, qkv, {B, S, C});
            Tensor f = tensor(T::INT32, fk, {B, S}), d = tensor(T::BF16, dqkv[2], {B, S, C}), g = tensor(T::BF16, dout, {B, S, O});
            Tensor s = tensor(T::BYTE, scratch, {(long)need});
            attention_forward(o, l, x, f, am[2], 0.125f, B, S, Nq, Nkv, HD, nullptr);
            attention_backward(d, g, o, l, x, f, s, 0.125f, B, S, Nq, Nkv, HD, nullptr);
        }
        if (hipDeviceSynchronize() != hipSuccess) std::exit(3);
        expect(equal(out[i], out[0], no * 2) && equal(lse[i], lse[0], nl * 4) && equal(dqkv[i], dqkv[0], nq * 2) && equal(am[i], am[0], 4), "attention");
    }
    const int N = 3, V = 9001, k = 4;
    const long P = 9004;
    std::vector<std::int32_t> tok = {5, 9000, -1};
    auto* t = static_cast<std::int32_t*>(device(tok.size() * 4, tok.data()));
    for (int bf = 0; bf < 2; ++bf) {
        std::vector<float> x32((std::size_t)N * P);
        std::vector<std::uint16_t> x16(x32.size());
        for (std::size_t i = 0; i < x32.size(); ++i) {
            r = r * 1664525u + 1013904223u;
            x16[i] = (std::uint16_t)(((r >> 16) & 0x81FFu) | 0x3F00u);
            const std::uint32_t bits = (std::uint32_t)x16[i] << 16;
            std::memcpy(&x32[i], &bits, 4);
        }
        const std::size_t size = bf ? 2 : 4, n = x32.size() * size;
        void* x = device(n, bf ? static_cast<const void*>(x16.data()) : x32.data());
        const std::size_t sn = get_token_logprobs_scratch_size(N, V, k);
        auto* s = static_cast<std::byte*>(device(sn));
        float* o[3];
        std::int32_t* ids[3];
        void* dx[3];
        for (int i = 0; i < 3; ++i) {   // logp, entropy, lse, top
            o[i] = static_cast<float*>(device((3 + k) * N * 4)), ids[i] = static_cast<std::int32_t*>(device(N * k * 4)), dx[i] = device(n);
            float *lp = o[i], *en = lp + N, *ls = en + N, *top = ls + N;
            if (i == 0) {
                auto f = [&](auto call, auto* logits) { llmq_detail::check(call(lp, en, ls, top, ids[0], logits, t, s, sn, N, V, P, k, nullptr)); };
                auto b = [&](auto call, auto* dl, auto* logits) { llmq_detail::check(call(dl, lp, en, logits, t, ls, en, nullptr, N, V, P, nullptr)); };
                if (bf) f(llmq_token_logprobs_bf16, (std::uint16_t*)x), b(llmq_token_logprobs_backward_bf16, (std::uint16_t*)dx[0], (std::uint16_t*)x);
                else f(llmq_token_logprobs_f32, (float*)x), b(llmq_token_logprobs_backward_f32, (float*)dx[0], (float*)x);
            } else if (i == 1) {
                if (bf) {
                    token_logprobs(lp, en, ls, top, ids[1], (const __hip_bfloat16*)x, t, s, sn, N, V, P, k, nullptr);
                    token_logprobs_backward((__hip_bfloat16*)dx[1], lp, en, (const __hip_bfloat16*)x, t, ls, en, nullptr, N, V, P, nullptr);
                } else {
                    token_logprobs(lp, en, ls, top, ids[1], (const float*)x, t, s, sn, N, V, P, k, nullptr);
                    token_logprobs_backward((float*)dx[1], lp, en, (const float*)x, t, ls, en, nullptr, N, V, P, nullptr);
                }
            } else {
                const T ty = bf ? T::BF16 : T::FP32;
                Tensor a = tensor(T::FP32, lp, {N}), e = tensor(T::FP32, en, {N}), l = tensor(T::FP32, ls, {N}), tp = tensor(T::FP32, top, {N, k});
                Tensor id = tensor(T::INT32, ids[2], {N, k}), lg = tensor(ty, x, {N, P}), tk = tensor(T::INT32, t, {N}), sc = tensor(T::BYTE, s, {(long)sn});
                Tensor d = tensor(ty, dx[2], {N, P});
                token_logprobs(a, e, l, tp, id, lg, tk, sc, N, V, P, k, nullptr);
                token_logprobs_backward(d, a, e, lg, tk, l, e, nullptr, N, V, P, nullptr);
            }
            if (hipDeviceSynchronize() != hipSuccess) std::exit(3);
            expect(equal(o[i], o[0], (3 + k) * N * 4) && equal(ids[i], ids[0], N * k * 4) && equal(dx[i], dx[0], n), bf ? "token_logprobs bf16" : "token_logprobs fp32");
        }
    }
}

int main(int argc, char** argv) {
    refusals();
    if (argc < 2 || std::strcmp(argv[1], "host") != 0) calls();
    std::printf("RESULT: %s\n", failures ? "FAIL" : "PASS");
    return failures != 0;
}
