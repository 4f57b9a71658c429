// Which launches a call of et_kv_tables makes.
#pragma once

namespace et {

// Tables that one workgroup takes (one launch|two, no slots to speak of, us: 512 entries 4.4|6.2, 2048 5.5|6.1, 4096 6.6|6.3, of 512 sequences 7.7|9.2, 8192 9.8|6.3, 16384 16.1|6.4).
constexpr int kOneEntries = 4096, kOneSequences = 512;
// Rows whose slots that workgroup writes, and of a sequence the sequence's own; those of more have a launch of their own, a thread each.  By the workgroup that writes the tables|apart, us:
//   one workgroup: 512 entries, 1024 rows 4.5|5.7, 2048 5.1|5.8, 4096 6.1|5.8, 8000 8.1|5.8;  4096 entries, 512 rows 6.7|8.1, 4096 8.4|8.0, 32768 23.1|8.0, 262144 138|8.4
//   of a sequence: 8192 pages, 256 rows 9.8|10.7, 1024 10.2|11.2, 2048 10.9|11.2, 4096 12.4|11.2, 65536 62.9|11.3;  64 sequences of 2048 pages, 1024 rows 7.3|8.2, 2048 8.0|8.3, 8192 13.5|9.2;
//   512 of 8192 pages, 512 rows 17.6|19.1
constexpr int kOneRows = 3000, kManyRows = 2048;

inline bool tables_of_one_workgroup(int max_pages, int B) { return B <= kOneSequences && (long long)B * max_pages <= kOneEntries; }
inline bool slots_apart(int max_pages, int B, int n) { return tables_of_one_workgroup(max_pages, B) ? (long long)B * n > kOneRows : n > kManyRows; }

}  // namespace et
