// The dense and gated layers of f32 rows (dense.hpp).
#include "dense_ops.hpp"

template struct arcn::DenseOps<float>;
