// Which of a paged-cache handle's workspaces a call's parts go to: plain host code without a GPU call, which the CPU tests
// compile by itself.
#pragma once
#include <algorithm>
#include <vector>

namespace illp {

// Work of one stream, or of one capture of a stream, runs in order and shares a workspace; two of them never do, unless the
// caller has bound streams to the same one.
struct Workspaces {
  struct Claim {
    const void* stream;
    unsigned long long capture;   // 0: not captured
    int workspace;
  };
  struct Bound {
    const void* stream;
    int workspace;
  };
  int count = 0;
  std::vector<Claim> claims;   // (at most `count`: reserved with the handle)
  std::vector<Bound> bound;

  bool claimed(int w) const {
    return std::any_of(claims.begin(), claims.end(), [&](const Claim& c) { return c.workspace == w; });
  }
  // The workspace that a stream is bound to; -1: none.
  int bound_to(const void* stream) const {
    for (const Bound& b : bound)
      if (b.stream == stream) return b.workspace;
    return -1;
  }
  // The workspace of an unbound stream's calls outside captures (capture 0) or in one; -1: there is none left.
  int claim(const void* stream, unsigned long long capture) {
    for (const Claim& c : claims)
      if (c.stream == stream && c.capture == capture) return c.workspace;
    for (int w = 0; w < count; w++) {
      if (claimed(w) || std::any_of(bound.begin(), bound.end(), [&](const Bound& b) { return b.workspace == w; })) continue;
      claims.push_back({stream, capture, w});
      return w;
    }
    return -1;
  }
  // False: an unbound stream's calls hold the workspace, or the stream is bound to another.
  bool bind(const void* stream, int w) {
    const int now = bound_to(stream);
    if (now < 0 && !claimed(w)) bound.push_back({stream, w});
    return now == w || bound_to(stream) == w;
  }
  void forget(const void* stream) {
    claims.erase(std::remove_if(claims.begin(), claims.end(), [&](const Claim& c) { return c.stream == stream; }), claims.end());
    bound.erase(std::remove_if(bound.begin(), bound.end(), [&](const Bound& b) { return b.stream == stream; }), bound.end());
  }
  void clear() {
    claims.clear();
    bound.clear();
  }
};

}  // namespace illp
