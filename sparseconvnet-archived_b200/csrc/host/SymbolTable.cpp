#include "SymbolTable.h"

SymbolTable::SymbolTable(cudaMemStream &memStream, int nSymbols, int nFeatures, float scale, const float *values)
    : table(false, 0), nSymbols(nSymbols), nFeatures(nFeatures), scale(scale), memStream(memStream) {
  if (nSymbols < 1 || (long long)nSymbols * nFeatures > 0x7fffffffll) throw ScnException("SymbolTable: bad number of symbols");
  if (!values) throw ScnException("SymbolTable: the table's values are needed");
  table.hVector().assign(values, values + (size_t)nSymbols * nFeatures);
}
void SymbolTable::forwards(SpatiallySparseBatchInterface &input) {
  const int rows = input.nSpatialSites;
  if ((int)input.symbols.size() != rows || input.nFeatures != nFeatures) throw ScnException("SymbolTable: one symbol per input row is needed");
  if ((long long)rows * nFeatures > 0x7fffffffll) throw ScnException("SymbolTable: more than 2^31 features in one batch; use smaller batches");
  input.sub->features.copyToGPU();
  input.sub->features.resize(rows * nFeatures);
  scnSafeCall(scn_embedding_forward(table.dPtr(), SCN_F32, nSymbols, nFeatures, input.symbols.dPtr(), rows, scale, input.sub->features.dPtr(), SCN_F32,
                                    nFeatures, nullptr, memStream.stream));
}
void SymbolTable::backwards(SpatiallySparseBatchInterface &input) {
  const int rows = input.nSpatialSites;
  if ((int)input.sub->dfeatures.size() != rows * nFeatures) throw ScnException("SymbolTable: the input's gradient is missing");
  dtable.copyToGPU();
  dtable.resize(nSymbols * nFeatures);
  const size_t bytes = scn_embedding_backward_workspace_bytes(rows, nSymbols, nFeatures);
  scnSafeCall(scn_embedding_backward(input.symbols.dPtr(), rows, input.sub->dfeatures.dPtr(), SCN_F32, nFeatures, nSymbols, nFeatures, scale, 0, dtable.dPtr(),
                                     nullptr, memStream.deviceScratch(bytes), bytes, memStream.stream));
}
void SymbolTable::update(float learningRate, float momentum) {
  const int n = nSymbols * nFeatures;
  if ((int)Mtable.size() != n) {
    Mtable.copyToGPU();
    Mtable.resize(n);
    Mtable.setZero(memStream);
  }
  scnSafeCall(scn_sgd_update(table.dPtr(), Mtable.dPtr(), dtable.dPtr(), n, learningRate, momentum, 0, memStream.stream));
}
