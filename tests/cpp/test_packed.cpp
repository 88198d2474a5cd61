// test_packed.cpp -- the packed-prompt and shared-prefix members of the C++ host side (include/turboshimmy.hpp) on the
// GPU, each against its formula in 64 bits on the host.
//
// Built by tests/cpp/Makefile, run by tests/test_gpu_cpp_packed.py on a GPU.  Prints one line per test; exit status 0
// when all pass.
#include <hip/hip_runtime_api.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <functional>
#include <random>
#include <string>
#include <vector>

#include "turboshimmy.hpp"

extern "C" {
// oracle/ts_oracle.c
void or_quantize_row(const float *x, int hd, float *scale_out, uint32_t *words);
void or_dequantize_row(const uint32_t *words, int hd, float scale, float *out);
}

namespace ts = turboshimmy;

namespace {

struct Failure {
    std::string msg;
};
void require(bool ok, const std::string &msg) {
    if (!ok) throw Failure{msg};
}
void hip_ok(hipError_t e, const char *what) {
    if (e != hipSuccess) throw Failure{std::string(what) + ": " + hipGetErrorString(e)};
}

// A device array of T, filled from / read back to host vectors.
template <typename T>
struct Dev {
    T *p = nullptr;
    size_t n = 0;
    explicit Dev(size_t count) : n(count) { hip_ok(hipMalloc(&p, sizeof(T) * (n ? n : 1)), "hipMalloc"); }
    explicit Dev(const std::vector<T> &h) : Dev(h.size()) {
        hip_ok(hipMemcpy(p, h.data(), sizeof(T) * n, hipMemcpyHostToDevice), "hipMemcpy H2D");
    }
    Dev(const Dev &) = delete;
    Dev &operator=(const Dev &) = delete;
    ~Dev() { (void)hipFree(p); }
    std::vector<T> host() const {
        std::vector<T> h(n);
        hip_ok(hipDeviceSynchronize(), "hipDeviceSynchronize");
        hip_ok(hipMemcpy(h.data(), p, sizeof(T) * n, hipMemcpyDeviceToHost), "hipMemcpy D2H");
        return h;
    }
};

std::vector<float> normal(std::mt19937 &g, size_t n) {
    std::normal_distribution<float> nd(0.0f, 1.0f);
    std::vector<float> x(n);
    for (auto &e : x) e = nd(g);
    return x;
}

// theta_i of a scaled table.
double theta(int i, int rope_dim, double base, double factor, int l_train, double alpha, double beta) {
    const double t = std::pow(base, -2.0 * i / rope_dim);
    if (!(beta > alpha)) return t / factor;
    const double r = (l_train * t / (2.0 * M_PI) - alpha) / (beta - alpha), ramp = std::fmin(std::fmax(r, 0.0), 1.0);
    return t * ((1.0 - ramp) / factor + ramp);
}

// One head's q rotated (pairs 2i, 2i + 1) at a position.
std::vector<double> turned(const float *x, int hd, int pos, double base) {
    std::vector<double> y(hd);
    for (int i = 0; i < hd / 2; i++) {
        const double a = pos * theta(i, hd, base, 1.0, 0, 0.0, 0.0), c = std::cos(a), s = std::sin(a);
        y[2 * i] = x[2 * i] * c - x[2 * i + 1] * s;
        y[2 * i + 1] = x[2 * i] * s + x[2 * i + 1] * c;
    }
    return y;
}

// softmax(q k_j / sqrt(hd)) v_j over n keys: rows of k and v at k(j), v(j).
std::vector<double> attend(const std::vector<double> &q, int hd, int n, const std::function<const float *(int)> &k,
                           const std::function<const float *(int)> &v) {
    std::vector<double> x(n), o(hd, 0.0);
    double m = -1e300, l = 0.0;
    for (int j = 0; j < n; j++) {
        double d = 0.0;
        for (int e = 0; e < hd; e++) d += q[e] * k(j)[e];
        x[j] = d / std::sqrt((double)hd);
        m = std::fmax(m, x[j]);
    }
    for (int j = 0; j < n; j++) {
        const double p = std::exp(x[j] - m);
        l += p;
        for (int e = 0; e < hd; e++) o[e] += p * v(j)[e];
    }
    for (auto &e : o) e /= l;
    return o;
}

// Rows of unit variance (values below 5): scores off by 2^-18 and less (22 bits of every factor, f32 sums), the output
// by twice that of the largest value.
void expect_close(double got, double want, const std::string &what) {
    require(std::fabs(got - want) <= 5.0 * 0x1p-16, what + ": " + std::to_string(got) + " vs " + std::to_string(want));
}

void test_rope_apply() {
    const int n = 7, heads = 3, hd = 40, rd = 24, n_pos = 5000;
    std::mt19937 g(1);
    const auto x = normal(g, (size_t)n * heads * hd);
    const std::vector<int32_t> pos = {0, 4999, 17, 1, 2500, 4000, 3};
    const auto rope = ts::RopeTable::scaled(n_pos, rd, 1e5, 4.0, 1024, 1.0, 16.0, 1.25);
    Dev<float> dx(x), dy(x.size());
    Dev<int32_t> dp(pos);
    for (int layout : {(int)TS_ROPE_INTERLEAVED, (int)TS_ROPE_HALF}) {
        ts::rope_apply(rope, layout, TS_DTYPE_F32, dx.p, heads * hd, dp.p, n, heads, hd, dy.p, heads * hd);
        const auto y = dy.host();
        for (int t = 0; t < n; t++)
            for (int h = 0; h < heads; h++) {
                const float *a = &x[((size_t)t * heads + h) * hd], *b = &y[((size_t)t * heads + h) * hd];
                for (int i = 0; i < rd / 2; i++) {
                    const double w = pos[t] * theta(i, rd, 1e5, 4.0, 1024, 1.0, 16.0), c = 1.25 * std::cos(w), s = 1.25 * std::sin(w);
                    const int p = layout == TS_ROPE_HALF ? i : 2 * i, q = layout == TS_ROPE_HALF ? i + rd / 2 : 2 * i + 1;
                    // (table, products and sum each rounded once)
                    const double tol = 0x1p-21 * 1.25 * (std::fabs(a[p]) + std::fabs(a[q]));
                    require(std::fabs(b[p] - (a[p] * c - a[q] * s)) <= tol && std::fabs(b[q] - (a[p] * s + a[q] * c)) <= tol,
                            "rotated pair " + std::to_string(i));
                }
                for (int d = rd; d < hd; d++) require(a[d] == b[d], "dims past the rotated ones are copied");
            }
    }
}

void test_append_and_read() {
    const int S = 3, H = 2, hd = 64;
    const std::vector<int32_t> off = {1, 6, 6, 40};
    std::mt19937 g(2);
    const size_t row = (size_t)H * hd;
    const auto k = normal(g, 41 * row), v = normal(g, 41 * row);
    ts::KVCache kv = ts::KVCache::new_int4(2, H, hd, 48, S);
    Dev<float> dk(k), dv(v), rk(std::vector<float>(41 * row, 3.0f)), rv(std::vector<float>(41 * row, 3.0f));
    kv.append_packed(1, TS_DTYPE_F32, dk.p, row, dv.p, row, off.data(), nullptr);
    kv.increment_packed(off.data());
    require(kv.get_seq_len(0) == 5 && kv.get_seq_len(1) == 0 && kv.get_seq_len(2) == 34, "lengths after the prompts");
    kv.read_packed(1, nullptr, off.data(), TS_DTYPE_F32, rk.p, row, rv.p, row);
    const auto gk = rk.host(), gv = rv.host();
    std::vector<uint32_t> w(hd / 8);
    std::vector<float> want(hd);
    for (const auto *io : {&k, &v}) {
        const auto &got = io == &k ? gk : gv;
        for (size_t r = 0; r < 41 * (size_t)H; r++) {
            float scale = 0.0f;
            or_quantize_row(io->data() + r * hd, hd, &scale, w.data());
            or_dequantize_row(w.data(), hd, scale, want.data());
            const bool inside = r >= (size_t)H && r < 40 * (size_t)H;
            for (int d = 0; d < hd; d++) require(got[r * hd + d] == (inside ? want[d] : 3.0f), "row " + std::to_string(r));
        }
    }
    bool threw = false;
    try {
        const std::vector<int32_t> far = {0, 44, 44, 44};
        kv.append_packed(1, TS_DTYPE_F32, dk.p, row, dv.p, row, far.data(), nullptr);
    } catch (const ts::Error &e) {
        threw = e.code() == TS_ERR_OVERFLOW;
    }
    require(threw, "rows past the window throw");
}

void test_attn_prompt() {
    const int NH = 4, H = 2, hd = 64;
    const std::vector<int32_t> off = {0, 37, 38, 90};
    std::mt19937 g(3);
    const auto q = normal(g, (size_t)90 * NH * hd), k = normal(g, (size_t)90 * H * hd), v = normal(g, (size_t)90 * H * hd);
    Dev<float> dq(q), dk(k), dv(v), dout(q.size());
    require(ts::attn_prompt_workspace(TS_DTYPE_BF16, 90, H, hd) == 0, "16-bit rows need no scratch");
    const uint64_t bytes = ts::attn_prompt_workspace(TS_DTYPE_F32, 90, H, hd);
    Dev<uint8_t> ws(bytes);
    ts::attn_prompt(TS_DTYPE_F32, dq.p, NH * hd, dk.p, H * hd, dv.p, H * hd, off.data(), 3, NH, H, hd, dout.p, NH * hd, ws.p, bytes);
    const auto out = dout.host();
    for (int s = 0; s < 3; s++)
        for (int t = off[s]; t < off[s + 1]; t++)
            for (int h = 0; h < NH; h++) {
                const float *qr = &q[((size_t)t * NH + h) * hd];
                auto at = [&](const std::vector<float> &x) {
                    return [&, s, h](int j) { return &x[((size_t)(off[s] + j) * H + h / 2) * hd]; };
                };
                const auto want = attend({qr, qr + hd}, hd, t - off[s] + 1, at(k), at(v));
                for (int d = 0; d < hd; d++) expect_close(out[((size_t)t * NH + h) * hd + d], want[d], "token " + std::to_string(t));
            }
}

// A prefix, a chunk of new tokens and one token with its append, against both caches read back.
void test_shared_prefix() {
    const int S = 2, NH = 4, H = 2, hd = 64, P = 100, C = 3;
    const double base = 10000.0;
    std::mt19937 g(4);
    const auto rope = ts::RopeTable::scaled(160, hd, base);
    ts::KVCache pre = ts::KVCache::new_int4(1, H, hd, P), kv = ts::KVCache::new_int4(1, H, hd, 32, S);
    const size_t row = (size_t)H * hd;
    {
        Dev<float> dk(normal(g, P * row)), dv(normal(g, P * row));
        const std::vector<int32_t> off = {0, P};
        pre.append_packed(0, TS_DTYPE_F32, dk.p, row, dv.p, row, off.data(), &rope);
        pre.increment_packed(off.data());
        hip_ok(hipDeviceSynchronize(), "hipDeviceSynchronize");
    }
    kv.share_prefix(pre);
    require(kv.get_window_base(0) == (uint32_t)P && kv.get_window_base(1) == (uint32_t)P, "the batch continues the prefix");
    const std::vector<int32_t> whole = {0, P};
    Dev<float> pk(P * row), pv(P * row);
    pre.read_packed(0, nullptr, whole.data(), TS_DTYPE_F32, pk.p, row, pv.p, row);
    const auto hpk = pk.host(), hpv = pv.host();
    int len = 0;
    for (int n : {C, 1}) {
        const auto q = normal(g, (size_t)S * n * NH * hd), k = normal(g, S * n * row), v = normal(g, S * n * row);
        Dev<float> dq(q), dk(k), dv(v), dout(q.size());
        const uint64_t bytes = kv.shared_workspace_bytes(pre, NH, n);
        Dev<uint8_t> ws(bytes);
        if (n > 1) kv.append_quant(0, dk.p, dv.p, n, rope);
        kv.attn_shared(pre, 0, 0, n > 1 ? nullptr : dk.p, n > 1 ? nullptr : dv.p, dq.p, NH, n, rope, dout.p, ws.p, bytes);
        require(kv.increment(n).is_ok(), "increment");
        const auto out = dout.host();
        const std::vector<int32_t> own = {0, len + n, 2 * (len + n)};
        Dev<float> ok(own[2] * row), ov(own[2] * row);
        kv.read_packed(0, nullptr, own.data(), TS_DTYPE_F32, ok.p, row, ov.p, row);
        const auto hk = ok.host(), hv = ov.host();
        for (int s = 0; s < S; s++)
            for (int t = 0; t < n; t++)
                for (int h = 0; h < NH; h++) {
                    const size_t r = ((size_t)s * n + t) * NH + h;
                    auto at = [&](const std::vector<float> &p, const std::vector<float> &o) {
                        return [&, s, h](int j) {
                            return j < P ? &p[((size_t)j * H + h / 2) * hd] : &o[((size_t)(own[s] + j - P) * H + h / 2) * hd];
                        };
                    };
                    const auto want = attend(turned(&q[r * hd], hd, P + len + t, base), hd, P + len + t + 1, at(hpk, hk), at(hpv, hv));
                    for (int d = 0; d < hd; d++) expect_close(out[r * hd + d], want[d], "token " + std::to_string(t));
                }
        len += n;
    }
    bool threw = false;
    try {
        kv.share_prefix(pre);
    } catch (const ts::Error &e) {
        threw = e.code() == TS_ERR_INVALID;
    }
    require(threw, "share_prefix of sequences that hold keys throws");
}

}  // namespace

int main() {
    const std::pair<const char *, std::function<void()>> tests[] = {
        {"test_rope_apply", test_rope_apply},
        {"test_append_and_read", test_append_and_read},
        {"test_attn_prompt", test_attn_prompt},
        {"test_shared_prefix", test_shared_prefix},
    };
    int failed = 0;
    for (const auto &t : tests) {
        std::printf("%s ...\n", t.first);
        std::fflush(stdout);
        try {
            t.second();
            std::printf("PASS %s\n", t.first);
        } catch (const Failure &f) {
            std::printf("FAIL %s: %s\n", t.first, f.msg.c_str());
            failed++;
        } catch (const std::exception &e) {
            std::printf("FAIL %s: exception %s\n", t.first, e.what());
            failed++;
        }
        std::fflush(stdout);
    }
    return failed ? 1 : 0;
}
