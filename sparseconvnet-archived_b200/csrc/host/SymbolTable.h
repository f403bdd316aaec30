// A table in front of the first layer for inputs whose sites carry a code (a pen stroke's kind, a material, a label) instead of
// real features (no reference counterpart): row r of the input's features is scale * table[symbol r], and a training batch
// also learns the table.
#pragma once
#include "SpatiallySparseBatchInterface.h"

class SymbolTable {
public:
  vectorCUDA<float> table;  // [nSymbols x nFeatures]
  vectorCUDA<float> Mtable; // momentum of the SGD update
  vectorCUDA<float> dtable; // gradient of the last training step
  int nSymbols, nFeatures;
  float scale;
  cudaMemStream &memStream;
  SymbolTable(cudaMemStream &memStream, int nSymbols, int nFeatures, float scale, const float *values);
  // input.symbols -> input.sub->features.  A negative symbol gives a zero row (a sample's background row, say).
  void forwards(SpatiallySparseBatchInterface &input);
  // input.sub->dfeatures -> dtable
  void backwards(SpatiallySparseBatchInterface &input);
  void update(float learningRate, float momentum); // by the momentum SGD of the learnt layers
};
