#include "AdamW.h"
#include <cmath>

AdamW::AdamW(float beta1, float beta2, float eps, float weightDecay, float maxNorm, int stateBits)
    : beta1(beta1), beta2(beta2), eps(eps), weightDecay(weightDecay), maxNorm(maxNorm), stateBits(stateBits), step(0) {
  if (stateBits != 32 && stateBits != 8) throw ScnException("AdamW: states have 8 or 32 bits");
  if (!std::isfinite(weightDecay)) throw ScnException("AdamW: the weight decay must be finite");
  scn_adamw_scalars_t s; // the kernel's own checks of the other numbers
  const scn_adamw_t h = {0.0, beta1, beta2, eps, 1.0, maxNorm, 1, 0};
  scnSafeCall(scn_adamw_scalars(&h, &s));
}
AdamW::~AdamW() {
  for (auto &s : states) cudaFree(s.second.block);
}
void AdamW::update(const std::vector<LearntParameter> &parameters, float learningRate, int batchSize, cudaMemStream &memStream) {
  std::vector<scn_adamw_tensor_t> list;
  for (const LearntParameter &p : parameters) {
    const size_t n = p.w->size(), blocks = (n + SCN_ADAMW_BLOCK - 1) / SCN_ADAMW_BLOCK;
    if (p.gradient->size() != n) throw ScnException("AdamW: a gradient is missing (run backwards on a TRAINBATCH first)");
    if (n == 0) continue;
    const size_t each = (n * (stateBits == 8 ? 1 : sizeof(float)) + 255) / 256 * 256, scales = stateBits == 8 ? (blocks * sizeof(float) + 255) / 256 * 256 : 0;
    State &s = states[p.w];
    if (s.n != n) {
      if (s.block) cudaSafeCall(cudaFree(s.block));
      s = State();
      cudaSafeCall(cudaMalloc(&s.block, 2 * (each + scales)));
      cudaSafeCall(cudaMemsetAsync(s.block, 0, 2 * (each + scales), memStream.stream));
      s.n = n;
    }
    char *b = (char *)s.block;
    scn_adamw_tensor_t t = {};
    t.d_w = p.w->dPtr();
    t.d_g = p.gradient->dPtr();
    t.d_m = b;
    t.d_v = b + each;
    if (stateBits == 8) {
      t.d_m_scale = (float *)(b + 2 * each);
      t.d_v_scale = (float *)(b + 2 * each + scales);
    }
    t.n = (long long)n;
    t.weight_decay = p.decays ? weightDecay : 0.f;
    t.w_min = p.least;
    t.g_type = SCN_F32;
    list.push_back(t);
  }
  const scn_adamw_t h = {learningRate, beta1, beta2, eps, 1.0 / batchSize, maxNorm, step + 1, (unsigned)(step + 1)};
  float *norm = nullptr;
  if (maxNorm > 0) {
    const size_t bytes = scn_grad_norm_workspace_bytes();
    char *scratch = (char *)memStream.deviceScratch(bytes + sizeof(float));
    norm = (float *)(scratch + bytes);
    scnSafeCall(scn_grad_norm(list.data(), (int)list.size(), norm, scratch, bytes, memStream.stream));
  }
  scnSafeCall(scn_adamw_step(list.data(), (int)list.size(), &h, nullptr, norm, memStream.stream));
  ++step; // (not where a call above was refused)
}
