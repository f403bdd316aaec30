// Training by AdamW on a caller's stream that legacy-stream copies do not wait for: what is saved behind a step is that step's result, and
// weights loaded behind one are not overwritten by it.  Built and run by tests/test_gpu_learnt_inputs_streams.py on a B200; prints "ALL OK".
#include <cmath>
#include <cstdio>
#include <random>
#include <string>
#include <vector>
#include "NetworkInNetworkLayer.h"
#include "SparseConvNetCUDA.h"

#define CHECK(cond)                                                                   \
  do {                                                                                \
    if (!(cond)) { std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); return 1; } \
  } while (0)

static const int nSymbols = 11, nF = 3, nClasses = 5, samples = 64;

static SpatiallySparseBatch &fill(SparseConvNetCUDA &cnn) {
  const int S = cnn.inputSpatialSize;
  SpatiallySparseBatch &b = cnn.batchPool[0];
  cnn.prepareBatch(b);
  b.reset();
  b.type = TRAINBATCH;
  SpatiallySparseBatchInterface &in = b.interfaces[0];
  in.nFeatures = nF; in.spatialSize = S; in.featuresPresent.hVector() = range(nF);
  in.backpropErrors = true;
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
// Everything learnt, as the device has it once the stream is idle.
static std::vector<float> learnt(SparseConvNetCUDA &cnn) {
  cudaStreamSynchronize(cnn.memStream.stream);
  std::vector<float> all;
  const auto take = [&](vectorCUDA<float> &v) {
    const size_t at = all.size();
    all.resize(at + v.size());
    cudaMemcpy(all.data() + at, v.dPtr(), sizeof(float) * v.size(), cudaMemcpyDeviceToHost);
  };
  for (auto l : cnn.layers)
    if (auto n = dynamic_cast<NetworkInNetworkLayer *>(l)) { take(n->W); take(n->B); }
  take(cnn.symbolTable->table);
  return all;
}
static std::vector<float> file(const std::string &name) {
  std::ifstream f(name, std::ios::binary);
  std::string s((std::istreambuf_iterator<char>(f)), std::istreambuf_iterator<char>());
  return std::vector<float>((const float *)s.data(), (const float *)s.data() + s.size() / sizeof(float));
}

int main(int, char **argv) {
  const std::string base = std::string(argv[1]) + "/w";
  try {
    cudaStream_t stream;
    cudaSafeCall(cudaStreamCreateWithFlags(&stream, cudaStreamNonBlocking));
    SparseConvNetCUDA cnn(2, nF, nClasses, stream, 1, 2);
    cnn.addLeNetLayerMP(96, 3, 1, 2, 2, VLEAKYRELU, 0.0f);
    for (int width : {192, 288, 416}) cnn.addLeNetLayerMP(width, 2, 1, 2, 2, VLEAKYRELU, 0.0f);
    cnn.addLeNetLayerMP(512, 2, 1, 1, 1, VLEAKYRELU, 0.0f);
    cnn.addSoftmaxLayer();
    std::vector<float> start(nSymbols * nF);
    std::mt19937 gen(1);
    std::normal_distribution<float> nd(0.f, 1.f);
    for (float &x : start) x = nd(gen);
    cnn.useSymbols(nSymbols, 2.f, start.data());
    cnn.useAdamW();
    std::ofstream nof, nog;
    cnn.processBatch(fill(cnn), 0.01f, 0.f, nof, nog);
    for (int times = 0; times < 4; ++times) {
      const std::vector<float> before = learnt(cnn);
      cnn.processBatch(fill(cnn), 0.01f, 0.f, nof, nog);
      cnn.saveWeights(base, times, false); // (the backward pass and the step are still in the stream)
      const std::vector<float> after = learnt(cnn);
      CHECK(after != before);
      CHECK(file(base + "_epoch-" + std::to_string(times) + ".cnn") == after);
    }
    std::printf("OK saved\n");
    for (int times = 0; times < 4; ++times) {
      cnn.processBatch(fill(cnn), 0.01f, 0.f, nof, nog);
      cnn.loadWeights(base, times, false);
      CHECK(learnt(cnn) == file(base + "_epoch-" + std::to_string(times) + ".cnn"));
    }
    std::printf("OK loaded\n");
  } catch (const std::exception &e) {
    std::printf("FAILED with exception: %s\n", e.what());
    return 1;
  }
  std::printf("ALL OK\n");
  return 0;
}
