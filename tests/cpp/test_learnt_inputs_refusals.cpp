// What symbol inputs refuse through the C++ classes, and that a refused call leaves the network as it was.
// Built and run by tests/test_gpu_learnt_inputs_refusals.py on a B200; prints "ALL OK" and exits 0 on success.
#include <cmath>
#include <cstdio>
#include <random>
#include <string>
#include <vector>
#include "NetworkArchitectures.h"
#include "NetworkInNetworkLayer.h"
#include "SparseConvNetCUDA.h"

#define CHECK(cond)                                                                   \
  do {                                                                                \
    if (!(cond)) { std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); return 1; } \
  } while (0)

static const int nSymbols = 11, nF = 3, nClasses = 5, samples = 4;

// A batch of symbols, a site in every second cell or so; `errors`: whether the input asks for its gradient.
static SpatiallySparseBatch &fill(SparseConvNetCUDA &cnn, batchType type, bool errors) {
  const int S = cnn.inputSpatialSize;
  SpatiallySparseBatch &b = cnn.batchPool[0];
  cnn.prepareBatch(b);
  b.reset();
  b.type = type;
  SpatiallySparseBatchInterface &in = b.interfaces[0];
  in.nFeatures = nF; in.spatialSize = S; in.featuresPresent.hVector() = range(nF);
  in.backpropErrors = errors;
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
// Everything that the network has learnt.
static std::vector<std::vector<float>> learnt(SparseConvNetCUDA &cnn) {
  std::vector<std::vector<float>> all = {values(cnn, cnn.symbolTable->table)};
  for (auto l : cnn.layers)
    if (auto n = dynamic_cast<NetworkInNetworkLayer *>(l)) { all.push_back(values(cnn, n->W)); all.push_back(values(cnn, n->B)); }
  return all;
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

    { // 2^30 + 1 rows of 3 features: their number does not fit 32 bits
      SpatiallySparseBatchInterface &in = fill(cnn, TESTBATCH, false).interfaces[0];
      const int rows = in.nSpatialSites;
      int *symbols = in.symbols.dPtr();
      in.nSpatialSites = (1 << 30) + 1;
      in.symbols.borrowDevice(symbols, in.nSpatialSites); // (refused before anything is read)
      bool refused = false;
      try { cnn.symbolTable->forwards(in); } catch (const std::exception &e) { refused = std::string(e.what()).find("smaller batches") != std::string::npos; }
      CHECK(refused);
      in.nSpatialSites = rows;
      in.symbols.borrowDevice(symbols, rows);
      cnn.symbolTable->forwards(in);
      std::printf("OK too many features\n");
    }

    // a training batch that forgot to ask for its input's gradient is refused before anything learns, under either optimiser, also where
    // the gradient of an earlier batch is still there
    std::ofstream nof, nog;
    for (int optimiser = 0; optimiser < 2; ++optimiser) {
      if (optimiser) cnn.useAdamW();
      for (int times = 0; times < 2; ++times) {
        const auto before = learnt(cnn);
        bool refused = false;
        try { cnn.processBatch(fill(cnn, TRAINBATCH, false), 0.01f, 0.f, nof, nog); } catch (const std::exception &e) { refused = true; }
        CHECK(refused && learnt(cnn) == before && (!optimiser || cnn.adamW->step == times));
        cnn.processBatch(fill(cnn, TRAINBATCH, true), 0.01f, 0.f, nof, nog);
        const auto after = learnt(cnn);
        for (size_t i = 0; i < after.size(); ++i) CHECK(after[i] != before[i]);
      }
    }
    std::printf("OK no gradient\n");
  } catch (const std::exception &e) {
    std::printf("FAILED with exception: %s\n", e.what());
    return 1;
  }
  std::printf("ALL OK\n");
  return 0;
}
