// Prints whether launches may overlap the kernel before them (1) or not (0): see overlap_attribute.
#include <cstdio>

#include "elb_common.cuh"

int main() {
  const cudaLaunchAttribute at = elb::overlap_attribute();
  std::printf("%d\n", at.id == cudaLaunchAttributeProgrammaticStreamSerialization ? at.val.programmaticStreamSerializationAllowed : -1);
  return 0;
}
