// How a batch whose requests share pages is cut up for attention (csrc/prefix_plan.cu makes the plan, csrc/prefix_attention.cu and csrc/attention_simt.cu read it).
//
// A plan is one int32 array: a header of 16, then at the offsets that the header names
//   items      8 each: first token (an index into `tokens`), tokens, first key, one past the last key, request whose block table names the keys, 1 if the tokens' positions
//              bound what they see (a request's own keys), first row of its results, first token of the batch if the others follow it one by one (else -1)
//   tokens     2 each: a token of the batch, its position
//   starts     by token of the batch (and one more): where its results are listed
//              (an item of few rows and several tiles of keys may leave two results for a row, the second ones behind all the first)
//   results    the first rows of a token's results, in ascending order of the keys that they stem from
//   positions  by token of the batch
// A row is a (token, query head of the group); a token's `rep` rows stand one behind the other.  Results of key/value head g lie `rows` further on than those of head g - 1.
#pragma once

constexpr int PLAN_HEADER = 16, PLAN_ITEM = 8;
enum { PLAN_ITEMS = 0, PLAN_TOKENS = 1, PLAN_AT_ITEMS = 2, PLAN_AT_TOKENS = 3, PLAN_AT_STARTS = 4, PLAN_AT_RESULTS = 5, PLAN_AT_POSITIONS = 6, PLAN_ROWS = 7 };
enum { ITEM_TOKEN = 0, ITEM_TOKENS = 1, ITEM_KEY_LO = 2, ITEM_KEY_HI = 3, ITEM_REQUEST = 4, ITEM_OWN = 5, ITEM_ROW = 6, ITEM_FIRST = 7 };
