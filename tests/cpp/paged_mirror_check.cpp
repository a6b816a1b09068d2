// Drives the paged cache through the C++ mirror: three tokens of one sequence in, with rotation by the caller's tables, then a single one; outputs
// against sums in 64 bits.  Prints "ok"; without a GPU ("--no-gpu") the status that refuses the context.
#include <cmath>
#include <cstdio>
#include <cstring>

#include "lumen_b200.hpp"

namespace L = lumen_b200;

int main(int argc, char **argv) {
    if (argc > 1 && !std::strcmp(argv[1], "--no-gpu")) {
        try {
            L::Context ctx(0);
        } catch (const L::Error &e) {
            std::printf("Error code=%d\n", e.code);
            return e.code == LUMEN_ERR_CUDA ? 0 : 1;
        }
        return 0;
    }
    try {
        const size_t D = 64, H = 2, max_pos = 8;
        L::Context ctx(0);
        std::vector<float> cos(max_pos * D / 2), sin(max_pos * D / 2);
        for (size_t p = 0; p < max_pos; ++p)
            for (size_t i = 0; i < D / 2; ++i) {
                const double a = (double)p * std::pow(10000.0, -2.0 * (double)i / (double)D);
                cos[p * D / 2 + i] = (float)std::cos(a);
                sin[p * D / 2 + i] = (float)std::sin(a);
            }
        const auto rope = L::RotaryEmbedding::from_tables(ctx, D, max_pos, cos.data(), sin.data());
        L::PagePool pool(ctx, 4, 8, 1, D, LUMEN_F32);
        std::vector<std::vector<double>> keys, values;
        auto turned = [&](const float *x, size_t pos) {
            std::vector<double> y(D);
            for (size_t i = 0; i < D / 2; ++i) {
                const double a = x[i], b = x[i + D / 2], c = cos[pos * D / 2 + i], s = sin[pos * D / 2 + i];
                y[i] = a * c - b * s;
                y[i + D / 2] = b * c + a * s;
            }
            return y;
        };
        unsigned seed = 1;
        for (size_t past = 0, n = 3; past < 4; past += n, n = 1) {
            std::vector<float> rows(n * (H + 2) * D);
            for (float &x : rows) x = (float)((seed = seed * 1664525u + 1013904223u) >> 9) / 4194304.f - 1.f;
            const std::vector<float> zeros(n * H * D);
            const L::Tensor in = L::Tensor::from_array_no_grad(ctx, {n, (H + 2) * D}, rows.data()), q = L::Tensor::from_array_no_grad(ctx, {n, H, D}, zeros.data()),
                            out = L::Tensor::from_array_no_grad(ctx, {n, H, D}, zeros.data());
            const float *at = static_cast<const float *>(lumen_tensor_data(in.get()));
            L::PageBatch batch(pool, H, {(int32_t)n}, {(int32_t)(past + n)}, {2}, 1);
            L::paged_append(pool, batch, &rope, at, at + H * D, at + (H + 1) * D, (H + 2) * D, (H + 2) * D, lumen_tensor_data(q.get()));
            L::paged_attention(pool, batch, lumen_tensor_data(q.get()), 0.125f, lumen_tensor_data(out.get()), LUMEN_F32);
            const std::vector<float> got = out.data();
            for (size_t t = 0; t < n; ++t) {
                const float *row = rows.data() + t * (H + 2) * D;
                keys.push_back(turned(row + H * D, past + t));
                values.emplace_back(row + (H + 1) * D, row + (H + 2) * D);
                for (size_t h = 0; h < H; ++h) {
                    const std::vector<double> query = turned(row + h * D, past + t);
                    std::vector<double> sum(D, 0.0);
                    double total = 0.0;
                    for (size_t j = 0; j < keys.size(); ++j) {
                        double s = 0.0;
                        for (size_t e = 0; e < D; ++e) s += query[e] * keys[j][e];
                        const double w = std::exp(0.125 * s);
                        total += w;
                        for (size_t e = 0; e < D; ++e) sum[e] += w * values[j][e];
                    }
                    for (size_t e = 0; e < D; ++e)  // (numbers of at most 1: scores of at most 8 in 32 bits, then a mean of values)
                        if (!(std::fabs(got[(t * H + h) * D + e] - sum[e] / total) < 1e-5)) throw std::runtime_error("output differs");
                }
            }
        }
        bool refused = false;
        try {
            L::PageBatch(pool, H, {1}, {9}, {2}, 1);  // nine positions, one page of eight
        } catch (const L::Error &e) {
            refused = e.code == LUMEN_ERR_KV_OVERFLOW;
        }
        if (!refused) throw std::runtime_error("a table too short was not refused");
        std::shared_ptr<L::PageBatch> left;
        {  // a batch keeps the context that it was made in
            L::Context own(0);
            left = std::make_shared<L::PageBatch>(L::PagePool(own, 1, 8, 1, D, LUMEN_F32), H, std::vector<int32_t>{1}, std::vector<int32_t>{1}, std::vector<int32_t>{0}, 1);
        }
        left.reset();
        std::printf("ok\n");
        return 0;
    } catch (const std::exception &e) {
        std::fprintf(stderr, "paged_mirror_check failed: %s\n", e.what());
        return 1;
    }
}
