// launch_turns.h -- whose turn it is to run a one-launch kernel (plain C++, no
// HIP: the CPU tests compile it on its own).
//
// The workgroups of a one-launch kernel (batch-1 layer, expert FFN, matvec) wait
// for earlier ones of their own grid.  One such grid drains: its items are
// dispatched in order, so the earliest unfinished one is resident or next.  Two
// at once need not: each XCD may be full of waiting workgroups of one grid while
// the item that these wait for has no place on another XCD, full of the other
// grid's.  So the kernels of different streams take turns: a launch on a stream
// other than the latest one's waits, on the device, for an event behind that.
// While one stream makes all the calls no event is recorded at all; where the
// second one begins, the event is put behind all that the first has queued.
#pragma once

#include <algorithm>
#include <vector>

namespace fdm {

struct LaunchTurns {
  enum Step {
    kGo,           // nothing of another stream is in the way
    kWait,         // wait for the event
    kMarkAndWait,  // record the event on `last`, then wait for it
  };
  void* last = nullptr;  // the stream of the latest launch
  bool any = false;      // there was one that may still run
  bool marked = false;   // the event stands behind it
  std::vector<void*> streams;  // that have launched and were not released

  Step before(void* s) const { return !any || s == last ? kGo : marked ? kWait : kMarkAndWait; }
  // After the launch; true: the event is to be recorded on s now.
  bool after(void* s) {
    if (std::find(streams.begin(), streams.end(), s) == streams.end()) streams.push_back(s);
    any = true;
    last = s;
    return marked = streams.size() > 1;
  }
  // A stream whose work is done (its handle may be reused).
  void forget(void* s) {
    streams.erase(std::remove(streams.begin(), streams.end(), s), streams.end());
    if (last == s) any = marked = false;
  }
};

}  // namespace fdm
