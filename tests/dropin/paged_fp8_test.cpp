// The 8-bit paged-cache calls of include/kernel_warpper.h from ordinary C++: three
// requests served step by step (prompts in chunks, decoded tokens, an idle
// request), the first step launched, the others one captured graph replayed with
// other lengths.  Every step is checked against the formulas in double on what
// the GPU was given: keys and values against the rows written, rows read back
// against the codes and scales of the pages, attention against those.
//
// Bounds: a row is rounded to codes when it is written and again when its block's
// scale grows, which a step does at most once, so at most 5 times here; a rounding
// is off by 2^-4 of the value or, below the least normal code, by 2^-10 scales of
// that time, which are no more than the last one.  (1 + 2^-4)^5 - 1 = 0.355.  Keys
// carry fp32 steps below 2^-16 of their terms.  Read rows are exact.  Attention's
// weights are rounded once at most, the same in numerator and denominator, which
// moves o by at most 2^-8 (sum w |v| + |o|), and o once more; scores and
// exponentials stay below 2^-12 of a weight.  Prints one line per check; exit
// status 0 iff every one passes.
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <string>
#include <vector>

#include "kernel_warpper.h"

extern "C" {
uint16_t or_f32_to_bf16(float f);
float or_bf16_to_f32(uint16_t h);
}

namespace {

using toyinfer::bf16;

int g_failures = 0;

void hip_ok(hipError_t e, const char* what) {
    if (e != hipSuccess) {
        std::fprintf(stderr, "HIP error %s: %s\n", what, hipGetErrorString(e));
        std::exit(2);
    }
}

void report(bool ok, const std::string& label) {
    std::printf("[%s] %s\n", ok ? "PASS" : "FAIL", label.c_str());
    std::fflush(stdout);
    if (!ok) ++g_failures;
}

// Device memory of T; bf16 tensors travel as their bits.
template <typename T>
struct Dev {
    T* p = nullptr;
    size_t n;
    explicit Dev(size_t count) : n(count) { hip_ok(hipMalloc(reinterpret_cast<void**>(&p), sizeof(T) * n), "malloc"); }
    ~Dev() { (void)hipFree(p); }
    Dev(const Dev&) = delete;
    Dev& operator=(const Dev&) = delete;
    template <typename U>
    void put(const std::vector<U>& h) {
        static_assert(sizeof(U) == sizeof(T), "");
        hip_ok(hipMemcpy(p, h.data(), sizeof(T) * std::min(n, h.size()), hipMemcpyHostToDevice), "h2d");
    }
    template <typename U>
    std::vector<U> get() const {
        static_assert(sizeof(U) == sizeof(T), "");
        std::vector<U> h(n);
        hip_ok(hipMemcpy(h.data(), p, sizeof(T) * n, hipMemcpyDeviceToHost), "d2h");
        return h;
    }
};

// An e4m3 code's value.
double code_value(uint8_t c) {
    const int e = (c >> 3) & 15, m = c & 7;
    if ((c & 0x7f) == 0x7f) return NAN;
    const double x = e ? std::ldexp(8 + m, e - 10) : std::ldexp(m, -9);
    return c & 0x80 ? -x : x;
}

std::vector<uint16_t> normal(std::mt19937& g, size_t n, float std) {
    std::normal_distribution<float> dist(0.0f, std);
    std::vector<uint16_t> x(n);
    for (auto& v : x) v = or_f32_to_bf16(dist(g));
    return x;
}

// y = rotate(x / sqrt(mean x^2 + eps) * w): the row, and the size of its terms.
void norm_rope(const uint16_t* x, const std::vector<uint16_t>& w, const float* cos_sin, uint32_t d, double eps,
               std::vector<double>& y, std::vector<double>& terms) {
    double ss = 0;
    for (uint32_t i = 0; i < d; ++i) ss += std::pow((double)or_bf16_to_f32(x[i]), 2);
    const double inv = 1.0 / std::sqrt(ss / d + eps);
    y.resize(d);
    terms.resize(d);
    for (uint32_t i = 0; i < d / 2; ++i) {
        const double a = or_bf16_to_f32(x[i]) * inv * or_bf16_to_f32(w[i]);
        const double b = or_bf16_to_f32(x[i + d / 2]) * inv * or_bf16_to_f32(w[i + d / 2]);
        const double c = cos_sin[2 * i], s = cos_sin[2 * i + 1];
        y[i] = a * c - b * s;
        y[i + d / 2] = b * c + a * s;
        terms[i] = terms[i + d / 2] = (std::fabs(a) + std::fabs(b)) * (std::fabs(c) + std::fabs(s));
    }
}

// A cached value against the row y it stands for, after up to 5 roundings at scales
// up to the block's.
bool near_cached(double got, double y, double term, double scale) {
    return std::fabs(got - y) <= 0.355 * std::fabs(y) + 7 * std::ldexp(scale, -10) + 2 * std::ldexp(term, -16);
}

void serve(uint32_t hq, uint32_t hkv, uint32_t d, uint32_t ps, uint32_t window, uint32_t sinks) {
    const uint32_t batch = 3, rows = 64, pages = 30, blocks = 8, max_pos = 128, group = hq / hkv;
    const float eps = 1e-6f;
    const uint32_t news[][3] = {{40, 5, 0}, {17, 1, 33}, {1, 1, 1}, {1, 0, 20}, {1, 4, 1}};
    std::mt19937 g(hq * d + window + 1);
    // K and V pages in one array, a page of K beside one of V; invalid codes and
    // scales where nothing was written.
    const size_t page = toyinfer::paged_fp8_page_bytes(ps, hkv, d);
    const uint64_t stride = 2 * page;
    report(page == (size_t)hkv * (ps * d + ps / 16 * 4) + (16 - hkv * (ps / 16 * 4) % 16) % 16, "page bytes");
    Dev<uint8_t> caches(pages * stride);
    Dev<bf16> q((size_t)rows * hq * d), k((size_t)rows * hkv * d), v((size_t)rows * hkv * d), q_out(q.n), o(q.n);
    Dev<bf16> k_read((size_t)batch * max_pos * hkv * d), v_read(k_read.n), qw(d), kw(d);
    caches.put(std::vector<uint8_t>(caches.n, 0xff));
    uint8_t *const kc = caches.p, *const vc = caches.p + page;
    const auto qwb = normal(g, d, 1.0f), kwb = normal(g, d, 1.0f);
    qw.put(qwb);
    kw.put(kwb);
    std::vector<float> rope((size_t)max_pos * d);
    for (uint32_t t = 0; t < max_pos; ++t)
        for (uint32_t i = 0; i < d / 2; ++i) {
            const double a = t * std::pow(1e6, -2.0 * i / d);
            rope[(size_t)t * d + 2 * i] = (float)std::cos(a);
            rope[(size_t)t * d + 2 * i + 1] = (float)std::sin(a);
        }
    Dev<float> rope_d(rope.size());
    rope_d.put(rope);
    Dev<uint32_t> ctx(batch), fresh(batch), free_pages(pages), num_free(1), table(batch * blocks), start(batch + 1),
        lens_d(batch), positions(rows), slots(rows), status(2), all_start(batch + 1);
    std::vector<uint32_t> stack(pages);
    for (uint32_t i = 0; i < pages; ++i) stack[i] = (7 * i + 3) % pages;
    free_pages.put(stack);
    num_free.put(std::vector<uint32_t>{pages});
    table.put(std::vector<uint32_t>(table.n, 0));
    const size_t plan_bytes = toyinfer::paged_attention_plan_bytes(batch, rows, hq, hkv, d);
    const size_t ws_bytes = toyinfer::paged_attention_workspace_bytes(hq, hkv, d);
    Dev<uint8_t> plan(plan_bytes), ws(ws_bytes);
    hip_ok(hipMemset(ws.p, 0xff, ws_bytes), "memset");
    hip_ok(hipMemset(ws.p, 0, 4 * (hkv + 2)), "memset");
    hipStream_t stream;
    hip_ok(hipStreamCreate(&stream), "stream");
    auto launch = [&]() {
        toyinfer::paged_tables_u32(ctx.p, fresh.p, batch, free_pages.p, pages, num_free.p, ps, table.p, blocks, rows,
                                   start.p, lens_d.p, positions.p, slots.p, status.p, stream);
        toyinfer::paged_attention_plan(start.p, lens_d.p, batch, rows, ps, blocks, window, sinks, hq, hkv, d, plan.p,
                                       plan_bytes, stream);
        toyinfer::paged_qkv_prologue_fp8(q.p, k.p, v.p, qw.p, kw.p, rope_d.p, max_pos, positions.p, slots.p, rows, eps,
                                         q_out.p, kc, vc, pages, ps, stride, hq, hkv, d, stream);
        toyinfer::paged_attention_fp8(q_out.p, kc, vc, o.p, table.p, plan.p, plan_bytes, batch, rows, pages, ps, stride,
                                      blocks, window, sinks, hq, hkv, d, ws.p, ws_bytes, stream);
        toyinfer::paged_kv_read_fp8(kc, vc, table.p, all_start.p, lens_d.p, batch, batch * max_pos, k_read.p, v_read.p,
                                    pages, ps, stride, blocks, hkv, d, stream);
    };
    hipGraph_t graph = nullptr;
    hipGraphExec_t exec = nullptr;
    std::vector<uint32_t> lens(batch, 0);
    // What every token's key and value were: double rows, [request][position][head][d].
    std::vector<std::vector<double>> keys(batch), key_terms(batch), values(batch);
    uint32_t left = pages;
    for (int step = 0; step < 5; ++step) {
        const std::string label = "paged fp8 " + std::to_string(hq) + "/" + std::to_string(hkv) + " D=" +
                                  std::to_string(d) + " window " + std::to_string(window) + " step " +
                                  std::to_string(step) + (step ? " (graph)" : "");
        const auto qb = normal(g, q.n, 1.5f), kb = normal(g, k.n, 1.5f), vb = normal(g, v.n, 1.0f);
        q.put(qb);
        k.put(kb);
        v.put(vb);
        ctx.put(lens);
        fresh.put(std::vector<uint32_t>(news[step], news[step] + batch));
        std::vector<uint32_t> first(batch + 1, 0);  // every cached token of every request is read
        for (uint32_t b = 0; b < batch; ++b) first[b + 1] = first[b] + lens[b] + news[step][b];
        all_start.put(first);
        o.put(std::vector<uint16_t>(o.n, 0x4040));
        k_read.put(std::vector<uint16_t>(k_read.n, 0x4040));
        hip_ok(hipDeviceSynchronize(), "sync");
        if (step == 0) {
            launch();
        } else {
            if (!exec) {
                hip_ok(hipStreamBeginCapture(stream, hipStreamCaptureModeThreadLocal), "capture");
                launch();
                hip_ok(hipStreamEndCapture(stream, &graph), "end capture");
                hip_ok(hipGraphInstantiate(&exec, graph, nullptr, nullptr, 0), "instantiate");
            }
            hip_ok(hipGraphLaunch(exec, stream), "graph");
        }
        hip_ok(hipStreamSynchronize(stream), "sync");
        const auto st = status.get<uint32_t>(), qs = start.get<uint32_t>(), slot = slots.get<uint32_t>(),
                   tab = table.get<uint32_t>(), ln = lens_d.get<uint32_t>();
        const auto all = caches.get<uint8_t>();
        const auto qo = q_out.get<uint16_t>(), ob = o.get<uint16_t>(), kr = k_read.get<uint16_t>(),
                   vr = v_read.get<uint16_t>();
        bool tables_ok = st[1] == 0, written_ok = true, read_ok = true, attn_ok = true;
        uint32_t t = 0;
        std::vector<double> y, terms, score;
        for (uint32_t b = 0; b < batch; ++b) {
            const uint32_t n = news[step][b], before = lens[b], len = before + n;
            tables_ok = tables_ok && qs[b] == t && ln[b] == len;
            left -= (len + ps - 1) / ps - (before + ps - 1) / ps;
            for (uint32_t i = 0; i < n; ++i)
                for (uint32_t h = 0; h < hkv; ++h) {
                    const size_t row = ((size_t)(t + i) * hkv + h) * d;
                    norm_rope(&kb[row], kwb, &rope[(size_t)(before + i) * d], d, eps, y, terms);
                    keys[b].insert(keys[b].end(), y.begin(), y.end());
                    key_terms[b].insert(key_terms[b].end(), terms.begin(), terms.end());
                    for (uint32_t e = 0; e < d; ++e) values[b].push_back(or_bf16_to_f32(vb[row + e]));
                }
            // The pages' codes and scales, against what was written and what was read.
            std::vector<double> kd((size_t)len * hkv * d), vd(kd.size());
            for (uint32_t j = 0; j < len; ++j)
                for (uint32_t h = 0; h < hkv; ++h)
                    for (int which = 0; which < 2; ++which) {
                        const uint8_t* const rec = &all[tab[b * blocks + j / ps] * stride + which * page];
                        const uint32_t in = j % ps;
                        float scale;
                        std::memcpy(&scale, rec + (size_t)hkv * ps * d + 4 * (h * (ps / 16) + in / 16), 4);
                        int exponent;
                        written_ok = written_ok && std::frexp(scale, &exponent) == 0.5f;
                        for (uint32_t e = 0; e < d; ++e) {
                            const size_t i = ((size_t)j * hkv + h) * d + e;
                            const double x = code_value(rec[((size_t)h * ps + in) * d + e]) * scale;
                            (which ? vd : kd)[i] = x;
                            written_ok = written_ok && near_cached(x, (which ? values : keys)[b][i],
                                                                   which ? 0 : key_terms[b][i], scale);
                            read_ok = read_ok && or_bf16_to_f32((which ? vr : kr)[(size_t)first[b] * hkv * d + i]) == x;
                        }
                    }
            for (uint32_t i = 0; i < n; ++i, ++t) {
                const uint32_t p = before + i;
                for (uint32_t h = 0; h < hq; ++h) {
                    const uint16_t* const qr = &qo[((size_t)t * hq + h) * d];
                    double m = -INFINITY, sum = 0;
                    score.assign(p + 1, -INFINITY);
                    for (uint32_t j = 0; j <= p; ++j) {
                        if (window && p - j >= window && j >= sinks) continue;
                        const double* const key = &kd[((size_t)j * hkv + h / group) * d];
                        double s = 0;
                        for (uint32_t e = 0; e < d; ++e) s += (double)or_bf16_to_f32(qr[e]) * key[e];
                        score[j] = s / std::sqrt((double)d);
                        m = std::max(m, score[j]);
                    }
                    for (auto& s : score) sum += s = std::exp(s - m);
                    for (uint32_t e = 0; e < d; ++e) {
                        double x = 0, size = 0;
                        for (uint32_t j = 0; j <= p; ++j) {
                            const double vj = vd[((size_t)j * hkv + h / group) * d + e];
                            x += score[j] / sum * vj;
                            size += score[j] / sum * std::fabs(vj);
                        }
                        const double got = or_bf16_to_f32(ob[((size_t)t * hq + h) * d + e]);
                        attn_ok = attn_ok && std::fabs(got - x) <= std::ldexp(size + 2 * std::fabs(x), -8) * (1 + 1.0 / 64) +
                                                                       std::ldexp(size, -12);
                    }
                }
            }
            lens[b] = len;
        }
        tables_ok = tables_ok && qs[batch] == t && st[0] == left;
        for (uint32_t r = t; r < rows; ++r) {
            tables_ok = tables_ok && slot[r] == 0xffffffffu;
            for (size_t e = 0; e < (size_t)hq * d; ++e) attn_ok = attn_ok && ob[(size_t)r * hq * d + e] == 0x4040;
        }
        for (size_t i = (size_t)first[batch] * hkv * d; i < kr.size(); ++i) read_ok = read_ok && kr[i] == 0x4040;
        num_free.put(std::vector<uint32_t>{st[0]});
        report(tables_ok, label + " tables");
        report(written_ok, label + " written k, v");
        report(read_ok, label + " read back");
        report(attn_ok, label + " attention");
    }
    hip_ok(hipGraphExecDestroy(exec), "graph");
    hip_ok(hipGraphDestroy(graph), "graph");
    hip_ok(hipStreamDestroy(stream), "stream");
}

}  // namespace

int main() {
    int n = 0;
    if (hipGetDeviceCount(&n) != hipSuccess || n < 1) {
        std::fprintf(stderr, "no HIP device\n");
        return 2;
    }
    serve(16, 8, 128, 16, 0, 0);
    serve(6, 2, 64, 32, 24, 4);
    std::printf("%s: %d failure(s)\n", g_failures ? "FAILED" : "ALL PASS", g_failures);
    return g_failures ? 1 : 0;
}
