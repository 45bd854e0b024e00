// Order in which copies of rows between the sequences of a cache are made so that every row is read before it is written
// (host code, no CUDA).
//
// A copy takes rows [begin, end) of sequence src to the same rows of sequence dst; a sequence is written by one copy at
// most, read by any number.  The copies out of one sequence form a group: one read, several writes.  The group that reads a
// must come before the group that writes a, and there is one such group at most, so "must come before" is a function on
// groups: its graph is trees that run into cycles.  Groups without a predecessor are taken off first; what is left are plain
// cycles, which are opened by holding the first group's rows while the others run.  Groups that depend on each other make up
// one program; programs touch different sequences, or only read the same ones, and run side by side.
#pragma once
#include <cstdint>
#include <vector>

enum : int { COPY_LOAD = 0, COPY_STORE = 1, COPY_HOLD = 2, COPY_STORE_HELD = 3 };

struct CopyStep {
  int slot, begin, end, op;     // loads have no rows of their own: those of the program
};

struct CopyProgram {
  std::vector<CopyStep> steps;
  int lo, hi;                   // rows that any step names
};

enum : int { COPY_PLAN_OK = 0, COPY_PLAN_RANGE = 1, COPY_PLAN_TWICE = 2, COPY_PLAN_CYCLE = 3 };

// copies: [n][4] src, dst, begin, end.  `most`: steps that a program may have in one launch.  A longer one is cut between
// groups into programs that have to run one after the other: `out` is then in launch order, and out_serial tells for each
// program whether it continues the one before it.  Cycles cannot be cut.
inline int copy_plan(const int32_t* copies, int n, int n_seqs, int t_max, int most, std::vector<CopyProgram>& out, std::vector<char>& out_serial) {
  out.clear();
  out_serial.clear();
  std::vector<int> writer(n_seqs, -1), head(n_seqs, -1), next(n, -1);      // next: copies with the same source
  std::vector<int> sources;
  for (int i = n - 1; i >= 0; --i) {      // backwards: lists come out in the caller's order
    const int src = copies[4 * i], dst = copies[4 * i + 1], b = copies[4 * i + 2], e = copies[4 * i + 3];
    if (src < 0 || src >= n_seqs || dst < 0 || dst >= n_seqs || b < 0 || e < b || e > t_max) return COPY_PLAN_RANGE;
    if (b == e) continue;
    if (writer[dst] >= 0) return COPY_PLAN_TWICE;
    writer[dst] = src;                    // a copy onto itself counts as a write (another copy may not write there too)
    if (src == dst) continue;
    if (head[src] < 0) sources.push_back(src);
    next[i] = head[src];
    head[src] = i;
  }
  // after[a]: the source whose group must come behind that of a
  std::vector<int> after(n_seqs, -1), waits(n_seqs, 0), part(n_seqs, -1);
  for (const int a : sources)
    if (writer[a] >= 0 && writer[a] != a) {
      after[a] = writer[a];
      ++waits[after[a]];
    }
  // parts of the graph: every chain ends in a root or a cycle
  std::vector<std::vector<int>> order;    // of each part: sources as they are to run; a cycle's follow a -1
  int n_parts = 0;
  for (const int a : sources) {
    if (part[a] >= 0) continue;
    std::vector<int> chain;
    int b = a;
    while (b >= 0 && part[b] == -1) {
      part[b] = -2;
      chain.push_back(b);
      b = after[b];
    }
    const int p = b >= 0 && part[b] >= 0 ? part[b] : n_parts++;
    for (const int c : chain) part[c] = p;
  }
  order.resize(n_parts);
  std::vector<int> ready;
  std::vector<char> done(n_seqs, 0);
  for (size_t i = sources.size(); i-- > 0;)
    if (!waits[sources[i]]) ready.push_back(sources[i]);
  while (!ready.empty()) {
    const int a = ready.back();
    ready.pop_back();
    done[a] = 1;
    order[part[a]].push_back(a);
    if (after[a] >= 0 && --waits[after[a]] == 0) ready.push_back(after[a]);
  }
  for (const int a : sources)
    if (!done[a]) {
      order[part[a]].push_back(-1);
      for (int b = a; !done[b]; b = after[b]) {
        done[b] = 1;
        order[part[a]].push_back(b);
      }
    }

  auto fresh = [&](bool serial) -> CopyProgram& {
    out.push_back({{}, t_max, 0});
    out_serial.push_back(serial);
    return out.back();
  };
  for (int p = 0; p < n_parts; ++p) {
    CopyProgram* prog = &fresh(false);
    auto stores = [&](int src, int op) {
      for (int i = head[src]; i >= 0; i = next[i]) {
        if ((int)prog->steps.size() >= most) {
          if (op != COPY_STORE) return false;
          prog = &fresh(true);
          prog->steps.push_back({src, 0, 0, COPY_LOAD});
        }
        const int b = copies[4 * i + 2], e = copies[4 * i + 3];
        prog->steps.push_back({copies[4 * i + 1], b, e, op});
        prog->lo = b < prog->lo ? b : prog->lo;
        prog->hi = e > prog->hi ? e : prog->hi;
      }
      return true;
    };
    const std::vector<int>& o = order[p];
    for (size_t i = 0; i < o.size(); ++i) {
      if (o[i] < 0) {
        // a cycle: hold the rows of its first source, run the others, write what was held
        size_t end = i + 2, need = 1;
        while (end < o.size() && o[end] >= 0) ++end;
        for (size_t j = i + 1; j < end; ++j) {
          need += j > i + 1;
          for (int c = head[o[j]]; c >= 0; c = next[c]) ++need;
        }
        if ((int)need > most) return COPY_PLAN_CYCLE;
        if ((int)(prog->steps.size() + need) > most) prog = &fresh(true);
        prog->steps.push_back({o[i + 1], 0, 0, COPY_HOLD});
        for (size_t j = i + 2; j < end; ++j) {
          prog->steps.push_back({o[j], 0, 0, COPY_LOAD});
          stores(o[j], COPY_STORE);
        }
        stores(o[i + 1], COPY_STORE_HELD);
        i = end - 1;
        continue;
      }
      if ((int)prog->steps.size() + 2 > most) prog = &fresh(true);
      prog->steps.push_back({o[i], 0, 0, COPY_LOAD});
      stores(o[i], COPY_STORE);
    }
  }
  return COPY_PLAN_OK;
}
