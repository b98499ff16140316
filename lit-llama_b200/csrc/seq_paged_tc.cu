// Longer chunks: so far the few-row kernel takes them all.
#include "seq_paged_attn.cuh"

namespace b2l {
namespace paged {

bool many_takes(int, int, int) { return false; }
int many_launch(const Attn&, int, cudaStream_t) { return 0; }

}  // namespace paged
}  // namespace b2l
