// test_evict.cpp -- the eviction members of the C++ host side (include/turboshimmy.hpp) on the GPU: one run of weighed
// attention, eviction and tokens behind it, against its formula in 64 bits on the host.
//
// Built by tests/cpp/Makefile, run by tests/test_gpu_cpp_evict.py on a GPU.  Prints one line per test; exit status 0
// when all pass.
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <random>
#include <string>
#include <vector>

#include "turboshimmy.hpp"

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
    for (auto &v : x) v = nd(g);
    return x;
}

constexpr int H = 2, NH = 4, HD = 64, CAP = 200;
constexpr double kBase = 10000.0;

// One token's attention over rows 0 .. n - 1 of k and v [slots][H][HD], its q at position pos: out, and the
// probabilities of each kv head.
void attend(const float *q, int pos, int n, const std::vector<float> &k, const std::vector<float> &v, std::vector<double> &out,
            std::vector<double> &w) {
    out.assign(NH * HD, 0.0);
    for (int h = 0; h < NH; h++) {
        double x[HD];
        for (int i = 0; i < HD / 2; i++) {
            const double t = pos * std::pow(kBase, -2.0 * i / HD), a = q[h * HD + 2 * i], b = q[h * HD + 2 * i + 1];
            x[2 * i] = a * std::cos(t) - b * std::sin(t);
            x[2 * i + 1] = a * std::sin(t) + b * std::cos(t);
        }
        const int kv = h / (NH / H);
        std::vector<double> p(n);
        double top = -1e300, sum = 0.0;
        for (int j = 0; j < n; j++) {
            for (int d = 0; d < HD; d++) p[j] += x[d] * k[((size_t)j * H + kv) * HD + d];
            p[j] /= std::sqrt((double)HD);
            top = std::max(top, p[j]);
        }
        for (auto &e : p) sum += e = std::exp(e - top);
        for (int j = 0; j < n; j++) {
            w[(size_t)kv * CAP + j] += p[j] / sum;
            for (int d = 0; d < HD; d++) out[h * HD + d] += p[j] / sum * v[((size_t)j * H + kv) * HD + d];
        }
    }
}

// f32 arithmetic of about 20 roundings of scores below 32, twice in a probability
void expect_close(double got, double want, double size, const std::string &what) {
    if (!(std::fabs(got - want) <= 1e-4 * (size + std::fabs(want))))
        throw Failure{what + ": " + std::to_string(got) + ", not " + std::to_string(want)};
}

void test_weigh_and_evict() {
    std::mt19937 g(7);
    auto kv = ts::KVCache::new_int4(1, H, HD, CAP, 1);
    ts::RopeTable rope = ts::RopeTable::scaled(CAP, HD, kBase);
    const size_t row = (size_t)H * HD;
    constexpr int N = 150, T = 5, KEEP = 60, SINK = 2, RECENT = 8;
    Dev<float> k(normal(g, N * row)), v(normal(g, N * row)), w(std::vector<float>(kv.weights_count(), 0.0f));
    require(kv.weights_count() == (size_t)H * CAP && kv.slots_count(KEEP) == (size_t)H * KEEP, "counts");
    kv.append_quant(0, k.p, v.p, N, rope);
    require(kv.increment(N).is_ok(), "increment");
    // a chunk
    const auto q = normal(g, (size_t)T * NH * HD);
    Dev<float> dk(normal(g, T * row)), dv(normal(g, T * row)), dq(q), out((size_t)T * NH * HD);
    kv.append_quant(0, dk.p, dv.p, T, rope);
    Dev<uint8_t> ws(std::max(kv.weigh_workspace_bytes(NH, T), kv.weigh_workspace_bytes(NH)));
    kv.attn_weigh(0, nullptr, nullptr, dq.p, NH, T, rope, w.p, true, out.p, ws.p, ws.n);
    require(kv.increment(T).is_ok(), "increment");
    const std::vector<int32_t> all = {0, N + T};
    Dev<float> rk((N + T) * row), rv((N + T) * row);
    kv.read_packed(0, nullptr, all.data(), TS_DTYPE_F32, rk.p, row, rv.p, row);
    auto hk = rk.host(), hv = rv.host();
    std::vector<double> want_w(H * CAP, 0.0), want;
    const auto o = out.host();
    for (int t = 0; t < T; t++) {
        attend(&q[(size_t)t * NH * HD], N + t, N + t + 1, hk, hv, want, want_w);
        for (int i = 0; i < NH * HD; i++) expect_close(o[(size_t)t * NH * HD + i], want[i], 1.0, "chunk's output");
    }
    const auto hw = w.host();
    for (int i = 0; i < H * CAP; i++) expect_close(hw[i], want_w[i], 1e-6, "chunk's weights");
    // the choice, and the rows
    Dev<int32_t> slots(kv.slots_count(KEEP));
    kv.evict(w.p, KEEP, SINK, RECENT, slots.p);
    const auto at = slots.host();
    require(kv.get_seq_len(0) == (uint32_t)KEEP && kv.get_window_base(0) == N + T - KEEP, "length and window base");
    const std::vector<int32_t> kept = {0, KEEP};
    Dev<float> ck(KEEP * row), cv(KEEP * row);
    kv.read_packed(0, nullptr, kept.data(), TS_DTYPE_F32, ck.p, row, cv.p, row);
    auto nk = ck.host(), nv = cv.host();
    const auto nw = w.host();
    for (int h = 0; h < H; h++) {
        std::vector<int> order;
        for (int p = SINK; p < N + T - RECENT; p++) order.push_back(p);
        std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return hw[h * CAP + a] > hw[h * CAP + b]; });
        order.resize(KEEP - SINK - RECENT);
        for (int p = 0; p < SINK; p++) order.push_back(p);
        for (int p = N + T - RECENT; p < N + T; p++) order.push_back(p);
        std::sort(order.begin(), order.end());
        for (int j = 0; j < KEEP; j++) {
            require(at[h * KEEP + j] == order[j], "slots");
            require(nw[h * CAP + j] == hw[h * CAP + order[j]], "kept weights");
            for (int d = 0; d < HD; d++)
                require(nk[((size_t)j * H + h) * HD + d] == hk[((size_t)order[j] * H + h) * HD + d] &&
                            nv[((size_t)j * H + h) * HD + d] == hv[((size_t)order[j] * H + h) * HD + d],
                        "kept rows");
        }
        for (int j = KEEP; j < CAP; j++) require(nw[h * CAP + j] == 0.0f, "weights behind the kept ones");
    }
    // a token behind them, appended in the call
    const auto q1 = normal(g, NH * HD);
    Dev<float> tk(normal(g, row)), tv(normal(g, row)), tq(q1), tout(NH * HD);
    kv.attn_weigh(0, tk.p, tv.p, tq.p, NH, 1, rope, w.p, false, tout.p, ws.p, ws.n);
    const std::vector<int32_t> more = {0, KEEP + 1};
    Dev<float> mk((KEEP + 1) * row), mv((KEEP + 1) * row);
    kv.read_packed(0, nullptr, more.data(), TS_DTYPE_F32, mk.p, row, mv.p, row);
    std::vector<double> w1(H * CAP, 0.0);
    attend(q1.data(), N + T, KEEP + 1, mk.host(), mv.host(), want, w1);
    const auto o1 = tout.host(), hw1 = w.host();
    for (int i = 0; i < NH * HD; i++) expect_close(o1[i], want[i], 1.0, "token's output");
    for (int i = 0; i < H * CAP; i++) expect_close(hw1[i], nw[i] + w1[i], 1e-6, "token's weights");
    bool threw = false;
    try {
        kv.select_slots(w.p, KEEP, KEEP, 1, slots.p);
    } catch (const ts::Error &e) {
        threw = e.code() == TS_ERR_INVALID;
    }
    require(threw, "more protected slots than kept ones throw");
}

}  // namespace

int main() {
    try {
        test_weigh_and_evict();
        std::printf("PASS test_weigh_and_evict\n");
        return 0;
    } catch (const Failure &f) {
        std::printf("FAIL test_weigh_and_evict: %s\n", f.msg.c_str());
    } catch (const std::exception &e) {
        std::printf("FAIL test_weigh_and_evict: exception %s\n", e.what());
    }
    return 1;
}
