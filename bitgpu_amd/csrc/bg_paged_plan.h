// The host side of a paged batch: checks of what a caller hands over (rows, lengths, page lists) and the
// plan the kernels run by. Plain C++ (no HIP), so it is tested on the CPU.
//
// A batch is n_seqs sequences; sequence b holds lens[b] positions in pages of `page` slots, its last
// rows[b] of them new in this call. Attention over it is cut into segments, a segment being a run of
// positions in the same pages for all of its member rows:
//   shared    the sequences' page lists form a tree (a node: sequences that list the same pages so far);
//             every edge of it with two or more sequences is one segment, scanned once for the rows of
//             all of them. Only pages that every row of the member sees whole are shared, so no mask.
//   private   the rest of each sequence, causal
// and a segment into units: a tile of 128, 32 or 16 of its rows (row = (token, head of the kv head's
// group)) times a chunk of its positions, one unit a workgroup and kv head. A row that meets several units
// gets a partial (o, m, l) from each, joined by the merge kernel; a row of one unit is stored directly.
// Everything is chosen by sizes and types alone, with the kernels' measured costs (kind, chunk).
#pragma once

#include <stdint.h>
#include <stdio.h>

#include <algorithm>
#include <string>
#include <vector>

namespace bg {

// One workgroup's attention work, for every kv head. Positions [key0, key1) (key0 a multiple of 32) of
// the page list at pages[table]; rows rho0 .. rho0 + n_rho - 1 of the tokens at toks[tok].
struct PagedUnit {
  int kind;    // 0: 128 rows, 32 a wave, the positions staged through LDS for all four; 1, 2: 32 and 16 rows,
               // the four waves splitting the positions
  int tok;
  int rho0, n_rho;
  int table;
  int key0, key1;
  int mask0;   // positions below this are seen by every row of the unit
  int chunk;   // which chunk of its segment: the partial slot is the token's `part` + chunk
  int page[4]; // the pages of the first four tiles, with which a wave each begins (one load in the chain
               // less before its first keys are on their way)
  int pad[3];
};
struct PagedTok {
  int t;       // row of q and out
  int pos;     // attends positions <= pos
  int part;    // partial slot of the segment's first chunk; -1: the row's only unit, stored directly
  int pad;
};
struct PagedMerge {
  int t, part, n, pad;
};

constexpr int kMergeFew = 8;

struct PagedShape {
  int kv_heads, G, D, dtype, page, n_pages;
  int cus;
  int max_seqs, max_tokens, max_pages;  // what the batch's arrays hold

  // shared segments on one sequence's path at most (what is below them stays private)
  static constexpr int kLevels = 4;
  int max_toks() const { return max_tokens * (kLevels + 1); }
  // units: a segment's row tiles unsplit (of 32 rows and more, and 2 at most for the rest), and what a
  // split adds, up to 8 units a CU
  long max_units() const {
    return (long)max_toks() * G / 32 + 2L * (2L * max_seqs) + 8L * cus;
  }
};
// storage bytes of 32 values (bg_kv dtypes: 0 f32, 1 f16, 2 q8 with its scale)
inline int paged_bytes32(int dtype) { return dtype == 0 ? 128 : dtype == 1 ? 64 : 36; }

// whether there is a kernel of 128-row units (elsewhere the 32-row ones are faster at every size)
constexpr bool paged_has_many(int D, int dtype) { return dtype == 1 || (dtype == 0 && D == 256); }

// and a kernel of 16-row units whose page loads are nontemporal
constexpr bool paged_has_stream(int D, int dtype) { return D == 128 && dtype == 1; }

struct PagedPlan {
  std::vector<PagedUnit> units;
  std::vector<PagedTok> toks;
  std::vector<PagedMerge> merges;
  std::vector<int> pages;        // every sequence's page list, one after the other
  std::vector<int> dst;          // per token: page * page size + slot
  std::vector<int> v_single;     // tokens whose V row is stored alone
  std::vector<int> v_group;      // first tokens of 16 that fill 16 aligned slots
  int n_tokens = 0, n_parts = 0;
  int n_merge_few = 0;           // merges of at most kMergeFew partials (the first ones)
  int n_many = 0, n_mid = 0;     // units of 128 rows (the first) and of 32 (the next)
  int shared_segments = 0;
  bool stream_few = false;       // 16-row units read their pages once, over 64 MB a layer
  int64_t keys = 0;              // positions scanned, a segment's once (a kv head)
  int write_page = -1;           // a page whose new positions another sequence also lists (see below)
};

class PagedPlanner {
 public:
  // Fills `out`; "" or what is wrong with the arguments. table: [n_seqs][stride], the first
  // ceil(lens[b] / page) entries of row b are read. `seen` is scratch kept between calls.
  std::string build(const PagedShape& sh, int n_seqs, const int* rows, const int* lens, const int* table, int stride,
                    PagedPlan& out) {
    char msg[200];
    sh_ = sh;
    out_ = &out;
    if (n_seqs < 0 || n_seqs > sh.max_seqs) {
      snprintf(msg, sizeof(msg), "%d sequences in a batch of at most %d", n_seqs, sh.max_seqs);
      return msg;
    }
    const int P = sh.page;
    long tokens = 0, pages = 0;
    for (int b = 0; b < n_seqs; b++) {
      if (lens[b] < 0 || lens[b] > kMaxLen || rows[b] < 0 || rows[b] > lens[b]) {
        snprintf(msg, sizeof(msg), "sequence %d: %d new rows of %d positions", b, rows[b], lens[b]);
        return msg;
      }
      const int need = lens[b] / P + (lens[b] % P != 0);
      if (need > stride) {
        snprintf(msg, sizeof(msg), "sequence %d: %d positions need %d pages of %d, its list holds %d", b, lens[b], need, P, stride);
        return msg;
      }
      tokens += rows[b];
      pages += need;
    }
    if (tokens > sh.max_tokens || pages > sh.max_pages) {
      snprintf(msg, sizeof(msg), "%ld new rows and %ld pages in a batch of at most %d and %d", tokens, pages, sh.max_tokens, sh.max_pages);
      return msg;
    }
    // the page lists; ids checked before anything uses them
    out.pages.resize(pages);
    off_.assign(n_seqs + 1, 0);
    for (int b = 0; b < n_seqs; b++) {
      const int need = lens[b] / P + (lens[b] % P != 0);
      off_[b + 1] = off_[b] + need;
      if (need == 0) continue;
      const int* ids = table + (size_t)b * stride;
      int* to = out.pages.data() + off_[b];
      unsigned most = 0;
      for (int i = 0; i < need; i++) {
        to[i] = ids[i];
        most = std::max(most, (unsigned)ids[i]);
      }
      if (most < (unsigned)sh.n_pages) continue;
      int i = 0;
      while (ids[i] >= 0 && ids[i] < sh.n_pages) i++;
      snprintf(msg, sizeof(msg), "sequence %d: page %d of its list is %d, of %d", b, i, ids[i], sh.n_pages);
      return msg;
    }
    n_seqs_ = n_seqs;
    rows_ = rows;
    lens_ = lens;
    out.n_tokens = (int)tokens;
    append(out);
    attend(out);
    return "";
  }

 private:
  static constexpr int kMaxLen = 1 << 30;  // positions of one sequence: the arithmetic below stays in int

  struct Segment {
    int table, key0, key1;  // positions; key1 the most any row sees
    int tok, n_tok;
    int rows;               // n_tok * G
    bool shared;
    int chunks = 1, chunk_len = 0;
  };

  // Where the new rows go, and the check that no two of them, and no other sequence's positions, share a
  // slot: write_page is a page that one sequence writes while another (or itself, twice) lists it with
  // written positions. The append refuses such a batch; attention alone may read it.
  void append(PagedPlan& out) {
    const int P = sh_.page;
    out.dst.clear();
    out.v_single.clear();
    out.v_group.clear();
    out.write_page = -1;
    if ((int)stamp_.size() < sh_.n_pages) stamp_.resize(sh_.n_pages, 0);
    if (epoch_ > 0x7ffffff0) {
      std::fill(stamp_.begin(), stamp_.end(), 0);
      epoch_ = 0;
    }
    const int written = ++epoch_;
    int tok = 0;
    for (int b = 0; b < n_seqs_; b++) {
      if (!rows_[b]) continue;
      const int p0 = lens_[b] - rows_[b], p1 = lens_[b];
      for (int i = p0 / P; i <= (p1 - 1) / P; i++) {
        const int id = out.pages[off_[b] + i];
        if (stamp_[id] == written) out.write_page = id;
        stamp_[id] = written;
      }
      for (int p = p0; p < p1; p++) out.dst.push_back(out.pages[off_[b] + p / P] * P + p % P);
      int p = p0;
      while (p < p1) {
        if ((p & 15) == 0 && p + 16 <= p1) {
          out.v_group.push_back(tok + p - p0);
          p += 16;
        } else {
          out.v_single.push_back(tok + p - p0);
          p++;
        }
      }
      tok += rows_[b];
    }
    // a written page listed elsewhere so far that its written slots are read there
    if (tok) {
      for (int b = 0; b < n_seqs_; b++) {
        const int n = off_[b + 1] - off_[b], first = rows_[b] ? (lens_[b] - rows_[b]) / P : n;
        for (int i = 0; i < std::min(n, first); i++) {
          const int id = out.pages[off_[b] + i];
          if (stamp_[id] == written && reads_written(out, b, i, id)) out.write_page = id;
        }
      }
    }
  }
  // sequence b reads page id (entry i of its list): does it read a slot that some sequence writes?
  bool reads_written(const PagedPlan& out, int b, int i, int id) const {
    const int P = sh_.page, upto = std::min(P, lens_[b] - i * P);
    for (int c = 0; c < n_seqs_; c++) {
      if (!rows_[c]) continue;
      const int p0 = lens_[c] - rows_[c];
      for (int j = p0 / P; j <= (lens_[c] - 1) / P; j++)
        if (out.pages[off_[c] + j] == id && (b != c || j != i) && upto > std::max(0, p0 - j * P)) return true;
    }
    return false;
  }

  // a 128-row tile a sequence fills by itself gains nothing from other sequences' rows
  bool shares(int b) const { return rows_[b] > 0 && rows_[b] * sh_.G < 128; }

  void attend(PagedPlan& out) {
    out.units.clear();
    out.toks.clear();
    out.merges.clear();
    segs_.clear();
    out.shared_segments = 0;
    out.keys = 0;
    first_.assign(n_seqs_, 0);
    start_.assign(n_seqs_, 0);
    std::vector<int> members;
    int tok = 0;
    for (int b = 0; b < n_seqs_; b++) {
      first_[b] = tok;
      tok += rows_[b];
      if (shares(b)) members.push_back(b);
    }
    split(members, 0, 0, 0);
    for (int b = 0; b < n_seqs_; b++) {
      if (!rows_[b] || lens_[b] <= start_[b] * sh_.page) continue;
      Segment s;
      s.table = off_[b];
      s.key0 = start_[b] * sh_.page;
      s.key1 = lens_[b];
      s.tok = (int)out.toks.size();
      s.n_tok = rows_[b];
      s.rows = rows_[b] * sh_.G;
      s.shared = false;
      push_tokens(b);
      segs_.push_back(s);
    }
    // Few-row segments join the 32-row units of others rather than take a launch of their own (16
    // sequences of 300 positions behind 4,096 f16 25 -> 19 us, 24 of 600 behind 8,192 40 -> 30), but where
    // they are most of the work: the 16-row kernel moves their pages faster at head_dim 128 (32 of 4,000
    // behind 2,048 f16 105, joined 110, f32 209 / 238, q8 79 / 92).
    few_as_mid_ = false;
    bool mid = false;
    double few = 0;
    for (const Segment& s : segs_) {
      if (kind(s) == 1) mid = true;
      if (kind(s) == 2) few += (double)(s.key1 - s.key0) * sh_.kv_heads;
    }
    few_as_mid_ = mid && (sh_.D == 256 || few < 5e5);
    chunk();
    emit(out);
  }

  void push_tokens(int b) {
    for (int i = 0; i < rows_[b]; i++)
      out_->toks.push_back(PagedTok{first_[b] + i, lens_[b] - rows_[b] + i, -1, 0});
  }
  // pages of sequence b that all of its rows see whole
  int whole(int b) const { return (lens_[b] - rows_[b] + 1) / sh_.page; }

  // The tree below `members`, which list the same pages up to `depth`; those from `start` on are not yet
  // in a segment.
  void split(const std::vector<int>& members, int start, int depth, int level) {
    if (members.size() < 2 || level == PagedShape::kLevels) {
      for (int b : members) start_[b] = start;
      return;
    }
    const std::vector<int>& pages = out_->pages;
    std::vector<int> order(members);
    auto key = [&](int b) { return depth < whole(b) ? pages[off_[b] + depth] : -1; };
    std::stable_sort(order.begin(), order.end(), [&](int x, int y) { return key(x) < key(y); });
    for (size_t i = 0; i < order.size();) {
      size_t j = i + 1;
      const int id = key(order[i]);
      while (j < order.size() && key(order[j]) == id) j++;
      if (id < 0 || j - i < 2) {
        for (size_t m = i; m < j; m++) start_[order[m]] = start;
        i = j;
        continue;
      }
      const std::vector<int> cls(order.begin() + i, order.begin() + j);
      int end = whole(cls[0]);
      for (int b : cls) {
        int e = depth + 1;
        const int lim = std::min(end, whole(b));
        while (e < lim && pages[off_[b] + e] == pages[off_[cls[0]] + e]) e++;
        end = e;
      }
      // Worth a segment when the reads it saves outweigh the partials it adds: every row's o is
      // written and read once more.
      long rows = 0;
      for (int b : cls) rows += rows_[b];
      const long saved = (long)(cls.size() - 1) * (end - start) * sh_.page * 2 * (sh_.D / 32) * paged_bytes32(sh_.dtype);
      const long added = rows * sh_.G * 2 * sh_.D * 4;
      if (saved > added) {
        Segment s;
        s.table = off_[cls[0]];
        s.key0 = start * sh_.page;
        s.key1 = end * sh_.page;
        s.tok = (int)out_->toks.size();
        s.n_tok = (int)rows;
        s.rows = (int)rows * sh_.G;
        s.shared = true;
        for (int b : cls) push_tokens(b);
        segs_.push_back(s);
        out_->shared_segments++;
        split(cls, end, end, level + 1);
      } else {
        split(cls, start, end, level);
      }
      i = j;
    }
  }

  // A segment's kind of units. 128-row units stage their positions once for four waves and reach the
  // matrix cores' rate; 32-row ones need a quarter of the workgroups' partials for the same parallelism,
  // and take a batch's few-row segments into the same launch. Where both exist the work decides, rows x
  // positions x kv heads (us in all, 128-row / 32-row units. f16 at 128, 8 kv heads, 32 sequences of 4
  // heads behind 16,384 positions 54 / 45, behind 32,768 72 / 79, a prompt of 777 34 / 47, of 100 19 / 15;
  // f16 at 256, 4 kv heads, 64 behind 4,096 65 / 59, behind 16,384 116 / 135; f32 at 256, 32 of 4 heads
  // behind 2,048 54 / 37, 64 of 6 behind 4,096 138 / 227).
  int kind(const Segment& s) const {
    if (s.rows <= 16) return few_as_mid_ ? 1 : 2;
    if (!paged_has_many(sh_.D, sh_.dtype)) return 1;
    const double work = (double)s.rows * (s.shared ? s.key1 - s.key0 : s.key1 - s.key0 - s.n_tok / 2) * sh_.kv_heads;
    return work > (sh_.dtype == 0 ? 2e6 : !s.shared ? 3e6 : sh_.D == 128 ? 20e6 : 12e6) ? 0 : 1;
  }
  // the unit that takes a segment's rows from r0 on: its kind and rows. What whole tiles leave over goes to
  // the smallest kind that takes it at once.
  int unit_kind(const Segment& s, int r0) const {
    const int left = s.rows - r0, k = kind(s);
    return left <= 16 && !few_as_mid_ ? 2 : k == 0 && left <= 32 ? 1 : k;
  }
  static int unit_rows(int kind) { return kind == 0 ? 128 : kind == 1 ? 32 : 16; }
  // row tiles in all, and those of the segment's own kind
  int n_tiles(const Segment& s) const {
    int n = 0;
    for (int r0 = 0; r0 < s.rows; r0 += unit_rows(unit_kind(s, r0))) n++;
    return n;
  }
  int own_tiles(const Segment& s) const {
    const int w = unit_rows(kind(s)), rest = s.rows % w;
    return s.rows / w + (rest && unit_kind(s, s.rows - rest) == kind(s));
  }
  // a segment's 32-position tiles
  static int tiles(const Segment& s) { return (s.key1 - s.key0 + 31) / 32; }
  // n tiles in equal chunks of about `len`
  static void split_evenly(unsigned n, unsigned len, unsigned& chunks, unsigned& chunk_len) {
    chunks = 1;
    chunk_len = (n + 1) & ~1u;  // even: 64 positions a step
    if (n <= len) return;
    chunks = (n - 1) / len + 1;
    chunk_len = ((n + chunks - 1) / chunks + 1) & ~1u;
    chunks = (n - 1) / chunk_len + 1;
  }
  static void cut(Segment& s, long len) {
    unsigned chunks, chunk_len;
    split_evenly((unsigned)tiles(s), (unsigned)std::min(len, (long)kMaxLen), chunks, chunk_len);
    s.chunks = (int)chunks;
    s.chunk_len = (int)chunk_len;
  }

  // Chunk lengths, by kind (each is a launch): the candidate with the least estimated time, in us, from
  // what the kernels measure. A launch of no more units than workgroup slots takes its longest unit, one
  // of more the slots' share of the work and part of a unit for the uneven end. A unit costs its start (its
  // descriptor, rows and queries come one after the other) and its tiles; every row of a split or shared
  // segment a partial a chunk, written and read.
  void chunk() {
    // [kind][head_dim 128, 256][dtype]: workgroups a CU, us of a 32-position tile of one unit with all of
    // them at work, and alone on a CU. 16-row units: 5.6 TB/s, and a wave's latency.
    static const int kSlots[3][2][3] = {{{2, 2, 2}, {1, 1, 1}}, {{2, 2, 3}, {1, 1, 2}}, {{2, 3, 3}, {1, 2, 2}}};
    static const double kFull[2][2][3] = {{{0, 2.1, 0}, {11.2, 2.5, 0}}, {{2.5, 0.72, 0.89}, {4.2, 0.92, 2.0}}};
    static const double kAlone[2][2][3] = {{{0, 1.26, 0}, {11.2, 2.5, 0}}, {{1.26, 0.39, 0.56}, {4.2, 0.92, 1.4}}};
    for (int kd = 0; kd < 3; kd++) {
      const bool few = kd == 2;
      const int wide = sh_.D == 256, per_cu = kSlots[kd][wide][sh_.dtype];
      const double slots = std::max(1.0, (double)sh_.cus * per_cu);
      const double full = few ? 2.0 * (sh_.D / 32) * paged_bytes32(sh_.dtype) * 32 * slots / 5.6e6 : kFull[kd][wide][sh_.dtype];
      const double alone = few ? 0.5 : kAlone[kd][wide][sh_.dtype];
      const double start = kd == 0 ? 6 : kd == 1 ? 7 : 5;
      double work = 0;
      long longest = 1, tiles1 = 0;
      cuts_.clear();
      for (const Segment& s : segs_) {
        if (kind(s) != kd) continue;
        const int n = tiles(s), own = own_tiles(s);
        work += (s.shared ? n : n - s.n_tok / 64.0) * own * sh_.kv_heads;
        longest = std::max(longest, (long)n);
        tiles1 += own;
        cuts_.push_back(Cut{(unsigned)n, own, s.rows, s.shared ? s.rows : 0});
      }
      if (tiles1 == 0) continue;
      // Segments of one length are cut alike: one entry for all of them, and no division for those a
      // candidate leaves whole (plans of 64 / 256 / 1,024 sequences of up to 40 pages in all 29 -> 15, 117 ->
      // 56, 519 -> 228 us of one core; of up to 500 pages 85 -> 55, 325 -> 194, 1,363 -> 801).
      std::sort(cuts_.begin(), cuts_.end(), [](const Cut& x, const Cut& y) { return x.tiles < y.tiles; });
      size_t last = 0;
      for (size_t i = 1; i < cuts_.size(); i++) {
        if (cuts_[i].tiles == cuts_[last].tiles) {
          cuts_[last].own += cuts_[i].own;
          cuts_[last].rows += cuts_[i].rows;
          cuts_[last].shared_rows += cuts_[i].shared_rows;
        } else {
          cuts_[++last] = cuts_[i];
        }
      }
      cuts_.resize(last + 1);
      double best = 1e30;
      long best_len = longest;
      for (long len = kd == 0 && !wide ? 8 : 4; len < 2 * longest; len = len * 9 / 8 + 1) {
        long n_units = 0, n_rows = 0;
        unsigned most = 1;
        for (const Cut& c : cuts_) {
          unsigned chunks, chunk_len;
          split_evenly(c.tiles, (unsigned)len, chunks, chunk_len);
          n_units += (long)chunks * c.own;
          n_rows += chunks > 1 ? (long)chunks * c.rows : c.shared_rows;
          most = std::max(most, std::min(chunk_len, c.tiles));
        }
        const double units = (double)n_units * sh_.kv_heads, rows = (double)n_rows * sh_.kv_heads;
        double t;
        if (units <= slots) {
          const double rate = !few ? (units * per_cu <= slots ? alone : full) : std::max(alone, full * units / slots);
          t = start + most * rate;
        } else {
          t = work * full / slots + start * (1 + units / slots) + (few ? 0.15 : 0.5) * most * full;
        }
        t += rows * (sh_.D + 2) * 4 * (1 / 5.0e6 + 1 / 4.0e6);
        if (t < best) {
          best = t;
          best_len = len;
        }
      }
      for (Segment& s : segs_)
        if (kind(s) == kd) cut(s, best_len);
    }
    // as many units as the arrays hold
    for (;;) {
      long units = 0;
      for (const Segment& s : segs_) units += (long)s.chunks * n_tiles(s);
      if (units <= sh_.max_units()) return;
      for (Segment& s : segs_) cut(s, 2L * s.chunk_len);
    }
  }

  void emit(PagedPlan& out) {
    // partial slots: a token's parts are the chunks of the segments it is in, one after the other
    count_.assign(out.n_tokens, 0);
    for (const Segment& s : segs_)
      for (int i = 0; i < s.n_tok; i++) count_[out.toks[s.tok + i].t] += s.chunks;
    base_.assign(out.n_tokens, 0);
    // rows of at most eight partials first: the merge kernel takes the two groups differently
    int parts = 0;
    out.n_merge_few = 0;
    for (int t = 0; t < out.n_tokens; t++) {
      base_[t] = -1;
      if (count_[t] < 2) continue;
      base_[t] = parts;
      parts += count_[t];
      if (count_[t] <= kMergeFew) out.merges.push_back(PagedMerge{t, base_[t], count_[t], 0});
    }
    out.n_merge_few = (int)out.merges.size();
    for (int t = 0; t < out.n_tokens; t++)
      if (count_[t] > kMergeFew) out.merges.push_back(PagedMerge{t, base_[t], count_[t], 0});
    out.n_parts = parts;
    for (const Segment& s : segs_) {
      for (int i = 0; i < s.n_tok; i++) {
        PagedTok& k = out.toks[s.tok + i];
        k.part = base_[k.t];
        if (base_[k.t] >= 0) base_[k.t] += s.chunks;
      }
    }
    // units by kind (128, 32, 16 rows), the heaviest first
    cost_.clear();
    for (const Segment& s : segs_) {
      out.keys += s.key1 - s.key0;
      for (int c = 0; c < s.chunks; c++) {
        for (int r0 = 0, R; r0 < s.rows; r0 += R) {
          PagedUnit u{};
          u.kind = unit_kind(s, r0);
          R = unit_rows(u.kind);
          u.tok = s.tok;
          u.rho0 = r0;
          u.n_rho = std::min(R, s.rows - r0);
          u.table = s.table;
          u.chunk = c;
          u.key0 = s.key0 + c * s.chunk_len * 32;
          int lo = out.toks[s.tok + r0 / sh_.G].pos, hi = lo;
          if (!s.shared) hi = out.toks[s.tok + (r0 + u.n_rho - 1) / sh_.G].pos;  // rows in order of position
          u.key1 = std::min(s.key0 + (c + 1) * s.chunk_len * 32, s.shared ? s.key1 : hi + 1);
          if (u.key1 < u.key0) u.key1 = u.key0;
          u.mask0 = s.shared ? s.key1 : lo + 1;
          for (int w = 0; w < 4; w++) {
            const int key = std::max(u.key0, std::min(u.key0 + 32 * w, (u.key1 - 1) & ~31));
            u.page[w] = out.pages[s.table + std::min(key, s.key1 - 1) / sh_.page];
          }
          out.units.push_back(u);
          cost_.push_back((u.key1 - u.key0 + 31) / 32);
        }
      }
    }
    order_.resize(out.units.size());
    for (size_t i = 0; i < order_.size(); i++) order_[i] = (int)i;
    std::stable_sort(order_.begin(), order_.end(), [&](int a, int b) {
      const int ka = out.units[a].kind, kb = out.units[b].kind;
      return ka != kb ? ka < kb : cost_[a] > cost_[b];
    });
    sorted_.clear();
    out.n_many = out.n_mid = 0;
    for (int i : order_) {
      out.n_many += out.units[i].kind == 0;
      out.n_mid += out.units[i].kind == 1;
    }
    // 16-row units: pages of their own, or the rest of a segment whose other units read the same
    bool once = true;
    double bytes = 0;
    for (const Segment& s : segs_) {
      if (kind(s) == 2) bytes += (double)(s.key1 - s.key0) * sh_.kv_heads * 2 * (sh_.D / 32) * paged_bytes32(sh_.dtype);
      else if (own_tiles(s) < n_tiles(s)) once = false;
    }
    out.stream_few = once && bytes > 64e6;
    for (int i : order_) sorted_.push_back(out.units[i]);
    out.units.swap(sorted_);
  }

  bool few_as_mid_ = false;
  PagedShape sh_{};
  PagedPlan* out_ = nullptr;
  int n_seqs_ = 0;
  const int* rows_ = nullptr;
  const int* lens_ = nullptr;
  std::vector<int> off_, first_, start_, count_, base_, order_;
  std::vector<long> cost_;
  std::vector<PagedUnit> sorted_;
  std::vector<Segment> segs_;
  struct Cut {  // segments of `tiles` tiles: row tiles of their own kind, rows, and those of shared ones
    unsigned tiles;
    long own, rows, shared_rows;
  };
  std::vector<Cut> cuts_;
  std::vector<int> stamp_;
  int epoch_ = 0;
};

}  // namespace bg
