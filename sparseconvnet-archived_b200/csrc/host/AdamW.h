// Adam with decoupled weight decay over all of a network's learnt tensors (no reference counterpart: the reference trains
// by its momentum SGD, NetworkInNetworkLayer.cu:26-40, a kernel for each tensor).  SparseConvNetCUDA::useAdamW makes a
// training batch's backwards() leave the gradients and one update() follow them.
#pragma once
#include <map>
#include <vector>
#include "utilities.h"
#include "vectorCUDA.h"

// A tensor that a training step changes, with its gradient.  decays: weight decay applies (matrices and tables, not biases
// and slopes); least: the values are held at or above it (-INFINITY: no bound).
struct LearntParameter {
  vectorCUDA<float> *w, *gradient;
  bool decays;
  float least;
};

class AdamW {
public:
  float beta1, beta2, eps, weightDecay, maxNorm; // maxNorm 0: no clipping
  int stateBits;                                 // 32 or 8 (scn_adamw_tensor_t says what the 8 bits hold)
  long long step;                                // steps done
  AdamW(float beta1, float beta2, float eps, float weightDecay, float maxNorm, int stateBits);
  ~AdamW();
  AdamW(const AdamW &) = delete;
  AdamW &operator=(const AdamW &) = delete;
  // One step.  The gradients are sums over `batchSize` samples; the step takes their mean (and clips its norm).  A norm that is
  // not finite, where maxNorm is set, leaves the parameters and moments as they are (the step counts all the same).
  void update(const std::vector<LearntParameter> &parameters, float learningRate, int batchSize, cudaMemStream &memStream);

private:
  struct State {
    void *block = nullptr; // both moments, then the scales of 8-bit ones
    size_t n = 0;
  };
  std::map<const void *, State> states; // by the parameter's vector, which lives as long as its layer
};
