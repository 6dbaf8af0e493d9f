// How the CTAs of a cluster leave an exchange of asynchronous copies between their shared memories.  Without CUDA in it:
// a test runs it on the CPU, with threads for the CTAs.
#pragma once

#ifdef __CUDACC__
#define B200_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define B200_HOST_DEVICE inline
#endif

namespace b200 {

// Every CTA sends its copies, waits (with a limit) for those sent to it, and calls this; `received`: they are all there.
// The cluster's barrier alone holds a CTA until every copy has been issued, not until it has landed: where a wait ran out, a
// peer that is later still may issue its copy just before it arrives, and the copy would be written into, and read
// from, memory that both have left and another kernel may own.  So a CTA that misses copies tells the others in front of
// the barrier; behind it the copies are certain to come and it waits for them, and a second barrier holds senders and
// receivers until then.  (Where nothing is missing every copy has landed, and one barrier is enough.)
template <typename Cluster>
B200_HOST_DEVICE void leave_exchange(Cluster& cluster, bool received) {
  if (!received) cluster.tell_late();
  cluster.barrier();
  if (cluster.any_late()) {
    cluster.wait_for_copies();
    cluster.barrier();
  }
}

}  // namespace b200
