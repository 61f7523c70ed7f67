// The host layer's one workspace holds what every prompt chunk and decode step of a context asks the library for. Sizes only: no GPU.
#include "attention_host.hpp"

#include <cmath>
#include <cstdio>
#include <random>

int main() {
    std::mt19937 rng(1);
    int wrong = 0;
    const int32_t heads[][3] = {{32, 8, 128}, {28, 4, 128}, {14, 2, 64}, {8, 8, 256}, {20, 20, 64}, {64, 8, 64}, {4, 1, 128}, {48, 48, 128}};
    for (const auto & h : heads)
        for (int32_t n_ctx : {16, 100, 128, 129, 300, 1000, 3000, 8192, 20000, 32768}) {
            dooms_amd::LlamaAttentionConfig c;
            c.n_layer = 1;
            c.n_ctx = n_ctx;
            c.n_head = h[0];
            c.n_head_kv = h[1];
            c.head_dim = h[2];
            const size_t bytes = dooms_amd::LlamaAttention::workspace_bytes(c);
            mx_attn_desc d{};
            d.n_head = c.n_head;
            d.n_head_kv = c.n_head_kv;
            d.head_dim = c.head_dim;
            d.q_stride = (c.n_head + 2 * c.n_head_kv) * c.head_dim;
            d.kv_stride = c.n_head_kv * c.head_dim;
            d.out_stride = c.n_head * c.head_dim;
            d.scale = 0.1f;
            for (int32_t rows = 1; rows <= n_ctx && rows <= 1024 * c.n_head_kv / c.n_head; rows++) {
                d.n_q = rows;
                d.causal = 1;
                for (int i = 0; i < 6; i++) {
                    d.p0 = i == 0 ? n_ctx - rows : i == 1 ? 0 : (int32_t)(rng() % (uint32_t)(n_ctx - rows + 1));
                    if (mx_attn_prefill_workspace_bytes(&d) > bytes) {
                        if (wrong++ < 5) std::fprintf(stderr, "%d/%d heads of %d, context %d: %d rows at %d need more\n", h[0], h[1], h[2], n_ctx, rows, d.p0);
                    }
                }
            }
            d.n_q = 1;
            d.causal = 0;
            for (int32_t len = 1; len <= n_ctx; len += 1 + n_ctx / 300)
                if (mx_attn_decode_workspace_bytes(&d, 1, len) > bytes) wrong++;
        }
    if (wrong) std::fprintf(stderr, "%d calls are short of workspace\n", wrong);
    return wrong != 0;
}
