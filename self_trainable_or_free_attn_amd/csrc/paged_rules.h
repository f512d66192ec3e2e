// How attention over paged caches cuts wide launches: the arithmetic of their lists of tiles, without GPU code, so that it can be
// compiled for the host as well.
//
// A list is the rows of a sequence (128 a tile, `group` rows a token) against its keys (64 a chunk). Under a causal mask its tiles
// read more chunks the later they stand. A tile of more than `piece` chunks is cut into as few pieces of about the same size as
// are not longer: one piece per started `piece`. Piece 0 of the tiles makes level 0, piece i level i; a level's tiles are the
// last ones of the list, so that tile and level follow from a number by counting.
#pragma once
#include "packed_rules.h"

namespace es {

// The tile that place y of a sequence falls into, whose tiles cost tile_cost each: one of them also for a y that no running counts
// give. (Counts that decrease name rows twice, and their costs may pass 2^31: no row outside the tensors may follow from that.)
ES_RULE int place_in(int y, int tile_cost, int tiles) {
  const int place = y / tile_cost;
  return place < 0 || tiles < 1 ? 0 : place < tiles ? place : tiles - 1;
}

struct WideList {
  int rows, tiles, chunks;  // chunks that the last tile reads, the most
  int behind;               // new tokens less all tokens of the sequence: new token i sees i + 1 - behind keys, those that are held
  int first;                // chunks that the first tile reads, about
};
constexpr int WIDE_ROWS = 128, WIDE_KEYS = 64;

ES_RULE int at_least(int x, int y) { return x > y ? x : y; }
ES_RULE int at_most(int x, int y) { return x < y ? x : y; }

// The list of nq tokens against `held` keys of `len` tokens (held <= len); head: tokens whose rows stand in its first tile.
ES_RULE WideList wide_list(int rows, int nq, int len, int held, int head, bool causal) {
  WideList x;
  x.rows = rows;
  x.tiles = (rows + WIDE_ROWS - 1) / WIDE_ROWS;
  x.chunks = (held + WIDE_KEYS - 1) / WIDE_KEYS;
  x.behind = nq - len;
  x.first = causal ? at_most(at_least(head - x.behind, 0) / WIDE_KEYS + 1, x.chunks) : x.chunks;
  return x;
}

// Tiles that read at most c chunks: the first ones. (64 c + behind tokens see at most c chunks; their rows are fewer than `rows`.)
ES_RULE int tiles_within(const WideList& x, int group, bool causal, int c) {
  if (x.chunks <= c) return x.tiles;
  if (!causal || c < 0) return 0;
  return at_least(WIDE_KEYS * c + x.behind, 0) * group / WIDE_ROWS;
}

// Chunks a piece at most: a piece costs a start and a partial, more of both with more rows.
ES_RULE int piece_of(const WideList& x, int per) { return at_least(per, x.rows <= 32 ? 4 : 8); }
ES_RULE int pieces_of(int chunks, int piece) { return chunks <= piece ? 1 : (chunks + piece - 1) / piece; }

// Levels above 0 that all tiles have.
ES_RULE int full_levels(const WideList& x, bool causal, int piece) {
  const int most = causal ? at_most(x.chunks - 1, at_least(-x.behind, 0) / WIDE_KEYS) : x.chunks - 1;
  return most > 0 ? most / piece : 0;
}
// Pieces above level 0.
ES_RULE int later_pieces(const WideList& x, int group, bool causal, int piece) {
  if (x.chunks <= piece) return 0;
  const int full = full_levels(x, causal, piece);
  int n = full * x.tiles;
  for (int c = (full + 1) * piece; c < x.chunks; c += piece) n += x.tiles - tiles_within(x, group, causal, c);
  return n;
}

// The pieces of a list's tiles that read more than `above` chunks (below `piece`), numbered level by level, the last tiles first.
ES_RULE bool piece_at(const WideList& x, int group, bool causal, int piece, int above, int i, int& tile, int& level) {
  int count = x.tiles - tiles_within(x, group, causal, above);
  level = 0;
  if (i >= count) {
    i -= count;
    const int full = full_levels(x, causal, piece);
    if (i < full * x.tiles) {
      level = 1 + i / x.tiles;
      i -= (level - 1) * x.tiles;
    } else {
      i -= full * x.tiles;
      level = full + 1;
      for (int c = level * piece;; c += piece, ++level) {
        if (c >= x.chunks) return false;
        count = x.tiles - tiles_within(x, group, causal, c);
        if (i < count) break;
        i -= count;
      }
    }
  }
  tile = x.tiles - 1 - i;
  return tile >= 0;
}
// and back
ES_RULE int piece_number(const WideList& x, int group, bool causal, int piece, int above, int tile, int level) {
  int n = x.tiles - 1 - tile;
  if (level > 0) {
    const int full = full_levels(x, causal, piece);
    n += x.tiles - tiles_within(x, group, causal, above) + at_most(level - 1, full) * x.tiles;
    for (int i = full + 1; i < level; ++i) n += x.tiles - tiles_within(x, group, causal, i * piece);
  }
  return n;
}

// Partials, which only the pieces of cut tiles have, are numbered in the same order without the tiles that are whole: that of
// piece_number with `above` = piece. Of the piece with number i, of a list with `level0` pieces of level 0 and `cuts` cut tiles,
// which are the first of them:
ES_RULE int partial_number(int i, int level0, int cuts) { return i < level0 ? i : i - level0 + cuts; }
// All partials of a launch of `tiles` tiles that allows `later` pieces above level 0: a cut tile has one of those at least.
ES_RULE long long most_partials(long long tiles, long long later) { return (tiles < later ? tiles : later) + later; }

// A launch's time in chunks: `big` items of `size` chunks, of which the GPU holds 1 / inv_slots, and small ones that take `small`
// together: rounds of big ones, small ones in the places that the last round leaves and behind it. An item's start takes as long
// as `start` chunks, a merge of tiles that are cut too. `mean`: all chunks over all places; what a CU does beside an item that is
// longer than that ends before it, and the item goes faster from there (a chunk takes 2.1 us beside another workgroup and 1.3
// alone: ALONE less). Small items behind the big ones end a quarter of a size late. ALONE 0: five sequences of 1 to 2048 tokens
// over 2048 to 75600 keys 344 us instead of 340, others the same; 0.8: 2048 causal tokens 66 us instead of 61. The quarter left
// out: 2048 tokens 66, 256 to 512 tokens over 9000 keys and fewer 65 instead of 55.6, 4305 beside 6 over 13663 144 instead of 135;
// a whole size: the same as a quarter.
constexpr float ALONE = 0.38f;
ES_RULE float wide_time(float big, float size, float small, float mean, bool cut, float start, float inv_slots) {
  const float rounds = big * inv_slots, whole = ceilf(rounds), each = size + start;
  const float left = (whole - rounds) * each;  // a place
  const float more = small * inv_slots - left, over = size - mean;
  return whole * each + (more > 0.0f ? more + 0.25f * size : 0.0f) + (cut ? start : 0.0f) - (over > 0.0f ? ALONE * over : 0.0f);
}

}  // namespace es
