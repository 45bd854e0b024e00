// Order in which copies of rows between the sequences of a cache are made so that every row is read before it is written
// (host code, no CUDA).
//
// A copy takes rows [begin, end) of sequence src to the same rows of sequence dst; a sequence is written by one copy at
// most, read by any number.  The copies out of one sequence form a group: one read, several writes.  The group that reads a
// must come before the group that writes a, and there is one such group at most, so "must come before" is a function on
// groups: its graph is trees that run into cycles.  Groups without a predecessor are taken off first; what is left are plain
// cycles, which are opened by holding the first group's rows while the others run.  Groups that depend on each other make up
// one program; programs touch different sequences, or only read the same ones, and run side by side.  In this order no group writes
// what a later one reads, so that the reads of the next groups may go ahead of the writes of this one: they do, four at a time.
#pragma once
#include <cstdint>
#include <vector>

// op of a step: which of five values is loaded, COPY_STORE more for its store; the last value is what a cycle holds
constexpr int COPY_VALUES = 4, COPY_HELD = COPY_VALUES, COPY_STORE = 8;

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
    auto store = [&](int i, int value) {
      const int b = copies[4 * i + 2], e = copies[4 * i + 3];
      prog->steps.push_back({copies[4 * i + 1], b, e, COPY_STORE + value});
      prog->lo = b < prog->lo ? b : prog->lo;
      prog->hi = e > prog->hi ? e : prog->hi;
    };
    auto writes = [&](int src) {
      int k = 0;
      for (int i = head[src]; i >= 0; i = next[i]) ++k;
      return k;
    };
    // sources [from, to) of the order, as many as fit together; one that fits nowhere is read again where it is cut
    const std::vector<int>& o = order[p];
    auto run = [&](size_t from, size_t to, bool may_cut) {
      while (from < to) {
        const size_t upto = from + COPY_VALUES < to ? from + COPY_VALUES : to;
        int need = 0;
        size_t end = from;
        while (end < upto && need + 1 + writes(o[end]) <= most) need += 1 + writes(o[end++]);
        if (end == from) {
          prog = &fresh(true);
          prog->steps.push_back({o[from], 0, 0, 0});
          for (int i = head[o[from]]; i >= 0; i = next[i]) {
            if ((int)prog->steps.size() >= most) {
              prog = &fresh(true);
              prog->steps.push_back({o[from], 0, 0, 0});
            }
            store(i, 0);
          }
          ++from;
          continue;
        }
        if (may_cut && (int)prog->steps.size() + need > most) prog = &fresh(true);
        for (size_t k = from; k < end; ++k) prog->steps.push_back({o[k], 0, 0, (int)(k - from)});
        for (size_t k = from; k < end; ++k)
          for (int i = head[o[k]]; i >= 0; i = next[i]) store(i, (int)(k - from));
        from = end;
      }
    };
    for (size_t i = 0; i < o.size();) {
      size_t end = i + (o[i] < 0);
      while (end < o.size() && o[end] >= 0) ++end;
      if (o[i] >= 0) {
        run(i, end, true);
      } else {
        // a cycle: hold the rows of its first source, run the others, write what was held
        int need = 0;
        for (size_t k = i + 1; k < end; ++k) need += 1 + writes(o[k]);
        if (need > most) return COPY_PLAN_CYCLE;
        if ((int)prog->steps.size() + need > most) prog = &fresh(true);
        prog->steps.push_back({o[i + 1], 0, 0, COPY_HELD});
        run(i + 2, end, false);
        for (int k = head[o[i + 1]]; k >= 0; k = next[k]) store(k, COPY_HELD);
      }
      i = end;
    }
  }
  // a first program that was passed over has no steps
  for (size_t i = 0; i < out.size();) {
    if (out[i].steps.empty()) {
      if (i + 1 < out.size()) out_serial[i + 1] = out_serial[i];
      out.erase(out.begin() + i);
      out_serial.erase(out_serial.begin() + i);
    } else {
      ++i;
    }
  }
  return COPY_PLAN_OK;
}
