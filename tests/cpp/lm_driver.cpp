// Runs a language-model-shaped policy through the C++ host layer (host/talos_lm.hpp) and dumps raw f64 for the Python test.
// Usage: lm_driver <mode> <in.bin> <out.bin> <B> <S> <dim> <heads> <kv_heads> <ff> <vocab> <p> <seed> <step>
// in.bin (f64): x [B,S,dim], the block's parameters in parameters() order, norm_f weight and bias, head weight [dim,vocab] and bias, tokens, old_logp,
// ref_logp, adv, weights [B*S], key counts [B].  out.bin: logits, loss, log-probabilities of the tokens, x.grad, every parameter's grad in the same order.
// Or: lm_driver junction <in.bin> <out.bin> <rows> <dim> <p> <seed>: x + dropout(x) and its norm; in.bin: x, weight, bias, g_h, g_y.  out.bin: the gradients of x,
// weight and bias of sum(h g_h) + sum(y g_y), then, over the same nodes, of sum(h g_h) alone.
#include <cstdio>
#include <string>
#include <vector>

#include "../../talos-xii_b200/host/talos_lm.hpp"
using namespace talos;

static int junction(char** argv) {
  const size_t R = std::stoul(argv[4]), D = std::stoul(argv[5]); const double p = std::stod(argv[6]); const uint64_t seed = std::stoull(argv[7]);
  std::FILE* in = std::fopen(argv[2], "rb"); if (!in) return 3;
  auto read = [&](size_t n) { std::vector<double> v(n); if (std::fread(v.data(), sizeof(double), n, in) != n) throw Panic("short input"); return v; };
  Tensor x = Tensor::new_(read(R * D), {R, D});
  LayerNorm norm(D, 1e-5);
  norm.weight.set_data(read(D)); norm.bias.set_data(read(D));
  Tensor gh = Tensor::new_(read(R * D), {R, D}), gy = Tensor::new_(read(R * D), {R, D});
  std::fclose(in);
  std::FILE* f = std::fopen(argv[3], "wb"); if (!f) return 3;
  auto dump = [&](const Tensor& t) { const std::vector<double> v = t.grad_vec(); std::fwrite(v.data(), sizeof(double), v.size(), f); };
  auto hy = dropout_add_layernorm(x, x, norm, p, seed, 5);
  ((hy.first * gh).sum() + (hy.second * gy).sum()).backward();
  dump(x); dump(norm.weight); dump(norm.bias);
  for (const Tensor* t : {&x, &norm.weight, &norm.bias, &hy.first, &hy.second}) t->zero_grad();
  (hy.first * gh).sum().backward();
  dump(x); dump(norm.weight); dump(norm.bias);
  std::fclose(f);
  return 0;
}

int main(int argc, char** argv) {
  if (argc == 8 && std::string(argv[1]) == "junction") {
    try { return junction(argv); } catch (const std::exception& e) { std::fprintf(stderr, "%s\n", e.what()); return 1; }
  }
  if (argc < 14) { std::fprintf(stderr, "usage\n"); return 2; }
  try {
    Runtime::get().mode = std::stoi(argv[1]);
    std::FILE* in = std::fopen(argv[2], "rb"); if (!in) return 3;
    const size_t B = std::stoul(argv[4]), S = std::stoul(argv[5]), D = std::stoul(argv[6]), H = std::stoul(argv[7]), Hk = std::stoul(argv[8]), ff = std::stoul(argv[9]), V = std::stoul(argv[10]);
    const double p = std::stod(argv[11]); const uint64_t seed = std::stoull(argv[12]), step = std::stoull(argv[13]);
    auto read = [&](size_t n) { std::vector<double> v(n); if (std::fread(v.data(), sizeof(double), n, in) != n) throw Panic("short input"); return v; };
    LmBlock block(D, H, Hk, ff, 1e-5, p, seed);
    LayerNorm norm_f(D, 1e-5); Linear head(D, V, true, seed + 9);
    Tensor x = Tensor::new_(read(B * S * D), {B, S, D});
    std::vector<Tensor> params = block.parameters();
    for (auto& t : norm_f.parameters()) params.push_back(t);
    for (auto& t : head.parameters()) params.push_back(t);
    for (auto& t : params) t.set_data(read(t.len()));
    const size_t n = B * S;
    auto ints = [](const std::vector<double>& v) { return std::vector<int32_t>(v.begin(), v.end()); };
    const std::vector<int32_t> tokens = ints(read(n));
    Tensor old = Tensor::new_(read(n), {n}), ref = Tensor::new_(read(n), {n}), adv = Tensor::new_(read(n), {n}), w = Tensor::new_(read(n), {n});
    const std::vector<int32_t> lens = ints(read(B));
    std::fclose(in);
    Tensor logits = head.forward(norm_f.forward(block.forward(x, step, &lens)));
    PolicyLossConfig cfg; cfg.clip_high = 0.28; cfg.c_kl = 0.05; cfg.c_entropy = 0.01;
    Tensor loss = policy_loss(logits, tokens, old, &ref, adv, &w, cfg, (double)n);
    loss.backward();
    std::FILE* f = std::fopen(argv[3], "wb"); if (!f) return 3;
    auto dump = [&](const std::vector<double>& v) { std::fwrite(v.data(), sizeof(double), v.size(), f); };
    dump(logits.to_vec()); dump(loss.to_vec()); dump(token_log_probs(logits, tokens).to_vec()); dump(x.grad_vec());
    for (auto& t : params) dump(t.grad_vec());
    std::fclose(f);
    Runtime::get().synchronize();
    return 0;
  } catch (const std::exception& e) { std::fprintf(stderr, "%s\n", e.what()); return 1; }
}
