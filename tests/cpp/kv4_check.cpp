// kv4_check — PageStack and PagedKv4Pool of solidattention/hip_kv.hpp on the
// GPU: two prompts, a decode step and the release, against attention in
// doubles over what the cache gives back.  Prints one JSON line; exit code 0
// when every bound holds.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <random>

#include "solidattention/hip_kv.hpp"

namespace hipkv = solidattention::hip;

namespace {

constexpr int kHeads = 2, kGroup = 2, kDim = 64;
constexpr float kScale = 0.125f;

std::vector<float> normal(std::mt19937& g, std::size_t n) {
  std::normal_distribution<float> d;
  std::vector<float> x(n);
  for (float& y : x) y = d(g);
  return x;
}

// The largest error of out [kHeads * kGroup][kDim] against softmax(q K) V over tokens [0, seen).
double worst(const float* q, const std::vector<float>& k, const std::vector<float>& v, std::size_t seen,
             const float* out) {
  double most = 0;
  for (int qh = 0; qh < kHeads * kGroup; ++qh) {
    const int h = qh / kGroup;
    std::vector<double> s(seen);
    for (std::size_t t = 0; t < seen; ++t)
      for (int c = 0; c < kDim; ++c) s[t] += double(q[qh * kDim + c]) * k[(t * kHeads + h) * kDim + c] * kScale;
    const double top = *std::max_element(s.begin(), s.end());
    double sum = 0;
    for (double& x : s) sum += x = std::exp(x - top);
    for (int c = 0; c < kDim; ++c) {
      double y = 0;
      for (std::size_t t = 0; t < seen; ++t) y += s[t] * v[(t * kHeads + h) * kDim + c];
      most = std::max(most, std::fabs(y / sum - out[qh * kDim + c]));
    }
  }
  return most;
}

}  // namespace

int main() {
  try {
    const std::vector<int32_t> lengths{75, 7};
    const int tokens = 82, row = kHeads * kDim, qrow = kHeads * kGroup * kDim;
    std::mt19937 g(1);
    hipkv::PagedKv4Pool pool(2, kHeads * kGroup, kHeads, 5, 9, kDim, tokens);
    hipkv::PageStack stack(9, 2, tokens);
    hipkv::DeviceArray<int32_t> count(2), status(1);
    hipkv::DeviceArray<float> k(tokens * row), v(tokens * row), q(tokens * qrow), out(tokens * qrow);
    count.upload(lengths);
    const std::vector<float> hk = normal(g, tokens * row), hv = normal(g, tokens * row), hq = normal(g, tokens * qrow);
    k.upload(hk), v.upload(hv), q.upload(hq);

    stack.reserve(pool.view(), count.get(), nullptr, nullptr, status.get());
    pool.store(k.get(), v.get(), SA_HIP_F32, stack.slots().get(), tokens, nullptr, status.get());
    pool.seal(0, nullptr, status.get());
    pool.prompt(q.get(), SA_HIP_F32, stack.query_start().get(), tokens, kScale, out.get(), nullptr, status.get());
    pool.load(k.get(), v.get(), SA_HIP_F32, stack.slots().get(), tokens, nullptr, status.get());
    const std::vector<float> held_k = k.download(), held_v = v.download(), got = out.download();
    double rounding = 0, prompt = 0;
    for (std::size_t i = 0; i < hk.size(); ++i)
      rounding = std::max(rounding, double(std::max(std::fabs(hk[i] - held_k[i]), std::fabs(hv[i] - held_v[i]))));
    std::vector<float> sk[2], sv[2];
    for (int b = 0, at = 0; b < 2; at += lengths[b++]) {
      sk[b].assign(held_k.begin() + at * row, held_k.begin() + (at + lengths[b]) * row);
      sv[b].assign(held_v.begin() + at * row, held_v.begin() + (at + lengths[b]) * row);
      for (int i = 0; i < lengths[b]; ++i)
        prompt = std::max(prompt, worst(&hq[(at + i) * qrow], sk[b], sv[b], i + 1, &got[(at + i) * qrow]));
    }

    hipkv::DeviceArray<int32_t> next(2);
    count.upload({1, 1});
    stack.reserve(pool.view(), count.get(), next.get(), nullptr, status.get());
    k.upload(hk), v.upload(hv);  // the first two rows are the step's tokens
    pool.append_seal(k.get(), v.get(), SA_HIP_F32, 0, nullptr, status.get());
    pool.decode(q.get(), SA_HIP_F32, kScale, out.get(), nullptr, nullptr, 0, 0, nullptr, status.get());
    pool.load(k.get(), v.get(), SA_HIP_F32, stack.slots().get(), 2, nullptr, status.get());
    const std::vector<float> new_k = k.download(), new_v = v.download(), step = out.download();
    double decode = 0;
    for (int b = 0; b < 2; ++b) {
      sk[b].insert(sk[b].end(), new_k.begin() + b * row, new_k.begin() + (b + 1) * row);
      sv[b].insert(sv[b].end(), new_v.begin() + b * row, new_v.begin() + (b + 1) * row);
      decode = std::max(decode, worst(&hq[b * qrow], sk[b], sv[b], lengths[b] + 1, &step[b * qrow]));
    }
    const bool counted = pool.seq_len().download() == std::vector<int32_t>{76, 8} &&
                         next.download() == std::vector<int32_t>{76, 8} &&
                         pool.sealed().download() == std::vector<int32_t>{2, 0} && stack.count().download()[0] == 5;
    count.upload({1, 1});
    stack.release(pool.view(), count.get(), nullptr, status.get());
    const bool released = stack.count().download()[0] == 9 && pool.seq_len().download() == std::vector<int32_t>{0, 0};
    const int flags = status.download()[0];
    bool refused = false;
    try {
      hipkv::PagedKv4Pool bad(1, 2, 2, 4, 4, 96);
    } catch (const std::runtime_error&) {
      refused = true;
    }
    std::printf("{\"rounding\": %.9g, \"prompt\": %.9g, \"decode\": %.9g, \"counted\": %s, \"released\": %s, "
                "\"refused\": %s, \"status\": %d}\n",
                rounding, prompt, decode, counted ? "true" : "false", released ? "true" : "false",
                refused ? "true" : "false", flags);
    // a code is half a scale off at most: (max - min) / 15 (1 + 2^-6) / 2, with |x| < 6 below 0.41, and the minimum's rounding
    return rounding <= 0.42 && prompt <= 1e-5 && decode <= 1e-5 && counted && released && refused && flags == 0 ? 0 : 1;
  } catch (const std::exception& e) {
    std::fprintf(stderr, "%s\n", e.what());
    return 2;
  }
}
