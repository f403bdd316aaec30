// Symbol inputs and AdamW through the C++ classes, as a program with its own batches uses them: interfaces filled by hand,
// SymbolTable::forwards(), layer by layer preprocess(), processBatch() on a TRAINBATCH, a layer's own backwards() beside it.
// Built and run by tests/test_gpu_learnt_inputs.py on a B200; prints "ALL OK" and exits 0 on success.
#include <cmath>
#include <cstdio>
#include <random>
#include <vector>
#include "NetworkArchitectures.h"
#include "NetworkInNetworkLayer.h"
#include "SparseConvNetCUDA.h"

#define CHECK(cond)                                                                   \
  do {                                                                                \
    if (!(cond)) { std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); return 1; } \
  } while (0)

static const int nSymbols = 11, nF = 3, nClasses = 5, samples = 4;

// The batch's interfaces 0: a site in every second cell or so, a symbol (row r: r % nSymbols, the background's negative) each.
static SpatiallySparseBatch &fill(SparseConvNetCUDA &cnn, batchType type) {
  const int S = cnn.inputSpatialSize;
  SpatiallySparseBatch &b = cnn.batchPool[0];
  cnn.prepareBatch(b);
  b.reset();
  b.type = type;
  SpatiallySparseBatchInterface &in = b.interfaces[0];
  in.nFeatures = nF; in.spatialSize = S; in.featuresPresent.hVector() = range(nF);
  in.backpropErrors = type == TRAINBATCH;
  std::mt19937 gen(3);
  std::vector<int> &symbols = in.symbols.hVector();
  symbols.clear();
  for (int i = 0; i < samples; ++i) {
    b.batchSize++;
    b.labels.hVector().push_back(i % nClasses);
    in.grids.push_back(SparseGrid());
    in.grids.back().backgroundCol = in.nSpatialSites++;
    symbols.push_back(-1);
    for (int k = 0; k < S * S; ++k)
      if (gen() % 2) {
        in.grids.back().mp[k] = in.nSpatialSites;
        symbols.push_back(in.nSpatialSites++ % nSymbols);
      }
  }
  cnn.symbolTable->forwards(in);
  in.uploadGrids(cnn.memStream);
  for (size_t i = 0; i < cnn.layers.size(); ++i) cnn.layers[i]->preprocess(b, b.interfaces[i], b.interfaces[i + 1]);
  return b;
}
static std::vector<float> values(SparseConvNetCUDA &cnn, vectorCUDA<float> &v) {
  cudaStreamSynchronize(cnn.memStream.stream);
  std::vector<float> copy = v.hVector();
  v.copyToGPU();
  return copy;
}
static bool finite(const std::vector<float> &v) {
  for (float x : v) if (!std::isfinite(x)) return false;
  return true;
}

int main() {
  try {
    SparseConvNet net(2, nF, nClasses);
    net.addLeNetLayerMP(32, 3, 1, 2, 2, VLEAKYRELU, 0.0f);
    net.addLeNetLayerMP(64, 2, 1, 1, 1, VLEAKYRELU, 0.0f);
    net.addSoftmaxLayer();
    SparseConvNetCUDA &cnn = *net.cnn;
    std::vector<float> start(nSymbols * nF);
    std::mt19937 gen(1);
    std::normal_distribution<float> nd(0.f, 1.f);
    for (float &x : start) x = nd(gen);
    cnn.useSymbols(nSymbols, 2.f, start.data());
    std::ofstream nof, nog;

    // the features are the table's scaled rows; a test batch learns nothing
    SpatiallySparseBatch &t = fill(cnn, TESTBATCH);
    std::vector<float> f = values(cnn, t.interfaces[0].sub->features);
    std::vector<int> codes = t.interfaces[0].symbols.hVector();
    CHECK(f.size() == codes.size() * nF);
    for (size_t r = 0; r < codes.size(); ++r)
      for (int c = 0; c < nF; ++c) CHECK(f[r * nF + c] == (codes[r] < 0 ? 0.f : 2.f * start[codes[r] * nF + c]));
    cnn.processBatch(t, 0, 0, nof, nog);
    CHECK(values(cnn, cnn.symbolTable->table) == start);
    std::printf("OK symbols\n");

    for (int bits : {32, 8}) {
      // AdamW: step 1 moves every value whose gradient is far above eps by the learning rate, whatever the gradient's size (m / sqrt(v)
      // is +-1 from its start at zero; 8 bits keep the sign and, in the first step, use the values before they are stored)
      cnn.useAdamW(0.9f, 0.999f, 1e-12f, 0.f, 0.f, bits);
      const std::vector<float> before = values(cnn, cnn.symbolTable->table);
      SpatiallySparseBatch &b = fill(cnn, TRAINBATCH);
      cnn.processBatch(b, 0.01f, 0.9f, nof, nog);
      const std::vector<float> after = values(cnn, cnn.symbolTable->table), g = values(cnn, cnn.symbolTable->dtable);
      CHECK(finite(after) && finite(g));
      int moved = 0;
      for (size_t i = 0; i < g.size(); ++i)
        if (std::fabs(g[i]) > 1e-6f) {
          // the step is 0.01 within a few roundings and eps / (|g| / 4) < 4e-6 of it, the new value within half a step of |w| < 8 (2.4e-7)
          CHECK(std::fabs(after[i] - before[i] + (g[i] > 0 ? 0.01f : -0.01f)) < 1e-6f);
          ++moved;
        }
      CHECK(moved > (int)g.size() / 2);

      // a layer's own backwards() behind it is what it always was: an update by momentum SGD of that layer alone
      NetworkInNetworkLayer *top = nullptr;
      size_t at = 0;
      for (size_t i = 0; i < cnn.layers.size(); ++i)
        if (auto n = dynamic_cast<NetworkInNetworkLayer *>(cnn.layers[i])) { top = n; at = i; }
      const std::vector<float> w = values(cnn, top->W);
      top->backwards(b, b.interfaces[at], b.interfaces[at + 1], 0.5f, 0.f);
      const std::vector<float> w1 = values(cnn, top->W);
      CHECK(finite(w1) && w != w1);
      top->weightsChanged();
      CHECK(values(cnn, cnn.symbolTable->table) == after);
    }
    std::printf("OK AdamW\n");

    // back to SGD: the table moves against its gradient
    cnn.useSGD();
    const std::vector<float> before = values(cnn, cnn.symbolTable->table);
    cnn.processBatch(fill(cnn, TRAINBATCH), 0.01f, 0.f, nof, nog);
    const std::vector<float> after = values(cnn, cnn.symbolTable->table), g = values(cnn, cnn.symbolTable->dtable);
    for (size_t i = 0; i < g.size(); ++i) CHECK(std::fabs(after[i] - (before[i] - 0.01f * g[i])) <= 4e-7f * (std::fabs(before[i]) + std::fabs(0.01f * g[i])));
    CHECK(before != after);
    std::printf("OK SGD\n");

    bool thrown = false;
    try {
      cnn.useAdamW();
      cnn.processBatch(fill(cnn, TRAINBATCH), NAN, 0.f, nof, nog);
    } catch (const std::exception &) { thrown = true; }
    CHECK(thrown && cnn.adamW->step == 0 && values(cnn, cnn.symbolTable->table) == after); // a refused step changes and counts nothing
  } catch (const std::exception &e) {
    std::printf("FAILED with exception: %s\n", e.what());
    return 1;
  }
  std::printf("ALL OK\n");
  return 0;
}
