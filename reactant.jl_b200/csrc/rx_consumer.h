// The stream of a consumer that was handed an array (DLPack), looked at when the consumer lets go of it.  The handle was
// kept since then and may mean another stream by now, or none: ids are never given out twice.  The queries are a parameter,
// so that the decision can be tested without a stream.
#pragma once

namespace rx {

enum class Consumer {
  Present,   // an event recorded on it covers its last use of the memory
  Captured,  // it is being captured into a graph: no event can be recorded until that has ended
  Gone       // there is nothing to record an event on: all work of the device is waited for
};
enum class Query { Ok, Implicit, Failed };  // Implicit: the legacy stream, while a stream that it waits for is captured

// queries.capturing(stream, &active) and queries.id(stream, &id), each a Query
template <class Queries, class Stream>
Consumer consumer_state(const Queries& queries, Stream stream, unsigned long long id) {
  bool active = false;
  const Query q = queries.capturing(stream, &active);
  if (q == Query::Failed) return Consumer::Gone;
  if (q == Query::Implicit || active) return Consumer::Captured;
  unsigned long long now = 0;
  return queries.id(stream, &now) == Query::Ok && now == id ? Consumer::Present : Consumer::Gone;
}

}  // namespace rx
