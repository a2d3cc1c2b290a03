// The decode operators through the C++ mirror (include/wgf/tensor.hpp): a small layer's prompt and one token.
#include <cmath>
#include <cstdio>
#include <cstring>

#include "wgf/tensor.hpp"

#define EXPECT(c)                                                               \
    do {                                                                        \
        if (!(c)) {                                                             \
            std::fprintf(stderr, "line %d: %s\n", __LINE__, #c);                \
            return 1;                                                           \
        }                                                                       \
    } while (0)

using wgf::Tensor;

int main(int argc, char** argv) {
    const bool dry = argc > 1 && !std::strcmp(argv[1], "--compile-only-device");
    wgf::Device dev(dry ? -1 : 0);
    constexpr int64_t H = 2, T = 70, D = 64;
    std::vector<float> ones(D, 1.f), k(H * T * D), cos(T * 2 * D / 2, 1.f), sin(T * 2 * D / 2, 0.f);
    for (size_t i = 0; i < k.size(); ++i) k[i] = (float)((int)(i * 7 % 255) - 127);
    Tensor<4, float> keys(dev, {1, H, T, D}, k.data());
    Tensor<1, float> w(dev, {D}, ones.data());
    Tensor<2, float> c(dev, {T * 2, D / 2}, cos.data()), s(dev, {T * 2, D / 2}, sin.data());

    wgf::KvCache<float> cache(dev, 1, H, D, T * 2);
    cache.append(keys, keys);
    EXPECT(cache.lengths()[0] == T);
    auto read = cache.read();
    EXPECT((read.first.shape() == std::array<int64_t, 4>{1, H, T, D}));
    auto last = Tensor<4, float>(keys).slice({{{0, 1}, {0, H}, {T - 1, T}, {0, D}}});
    auto turned = last.qk_norm_rope(last, w, w, c, s, 1e-5f, 3);
    auto q = cache.append_qk(last, last, last, w, w, c, s, 1e-5f);
    auto out = cache.attention(q, 0.125f);
    EXPECT(cache.lengths()[0] == T + 1);
    wgf::KvCache<float> same = cache;
    same.truncate({T});
    EXPECT(cache.lengths()[0] == T);
    bool refused = false;
    try {
        cache.truncate({T, T});
    } catch (const wgf::Error& e) {
        refused = e.code == WGF_ERR_SHAPE;
    }
    EXPECT(refused);

    const uint8_t codes[2] = {0x1f, 0x08};   // 15, 1, 8: 7, -7, 0 steps
    const float scale = 0.5f;
    auto q4 = wgf::Q4Weight::from_codes(dev, 1, 3, 32, codes, &scale);
    auto of = Tensor<2, float>(dev, {1, D}, ones.data()).quantize_q4(32);
    EXPECT(q4.rows() == 1 && q4.columns() == 3 && of.columns() == D);
    const float x[3] = {1.f, 2.f, 5.f};
    auto y = Tensor<2, float>(dev, {1, 3}, x).mat_mul_q4(q4);
    auto full = q4.dequantize<float>();
    if (dry) {
        y.materialize();
        std::printf("decode ok\n");
        return 0;
    }
    // keys are whole numbers up to 127 and every block has a 127 in it: the codes are the keys
    auto rk = read.first.as_slice();
    for (int64_t t = 0; t < T; ++t)
        for (int64_t d = 0; d < D; ++d) EXPECT((rk[{0, 1, t, d}] == k[(size_t)((T + t) * D + d)]));
    auto a = turned.first.as_slice(), b = turned.second.as_slice(), qq = q.as_slice();
    EXPECT(a == b && a == qq);
    for (int64_t d = 0; d < D; ++d) EXPECT((std::isfinite(out.as_slice()[{0, 0, 0, d}])));
    EXPECT((y.as_slice()[{0, 0}] == 3.5f - 7.f));
    auto f = full.as_slice();
    EXPECT((f[{0, 0}] == 3.5f && f[{0, 1}] == -3.5f && f[{0, 2}] == 0.f));
    std::printf("decode ok\n");
    return 0;
}
