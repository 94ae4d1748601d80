// What a captured step holds: its memset nodes, which are not safe in a graph without branches.
#include <cstdlib>

#include "common.h"

using namespace asrn;

extern "C" int64_t asrn_graph_memsets(void* graph) {
  size_t n = 0;
  if (!graph || hipGraphGetNodes((hipGraph_t)graph, nullptr, &n) != hipSuccess) {
    (void)hipGetLastError();                  // the calling thread's next launch check starts clean
    fail("asrn_graph_memsets: no graph");
    return -1;
  }
  if (n == 0) return 0;
  hipGraphNode_t* nodes = (hipGraphNode_t*)malloc(n * sizeof(hipGraphNode_t));
  bool ok = nodes && hipGraphGetNodes((hipGraph_t)graph, nodes, &n) == hipSuccess;
  int64_t found = 0;
  for (size_t i = 0; ok && i < n; ++i) {
    hipGraphNodeType type;
    ok = hipGraphNodeGetType(nodes[i], &type) == hipSuccess;
    found += ok && type == hipGraphNodeTypeMemset;
  }
  free(nodes);
  if (ok) return found;
  (void)hipGetLastError();
  fail("asrn_graph_memsets: the graph's nodes cannot be read");
  return -1;
}
