// Which elements of a tensor layer norm's copies take; host code too, so that it can be looked at without a device.
#pragma once

#ifdef __CUDACC__
#define FDA_NORM_COPY __host__ __device__ __forceinline__
#else
#define FDA_NORM_COPY inline
#endif

namespace fda_norm {

// Elements from the first of a row to the tensor's end, `left` rows from this one on (none behind the last); only as many of them as make a
// difference to a copy of that row.
FDA_NORM_COPY int room_of(long long left, int width, int each) {
    return left <= 0 ? 0 : (left <= each ? (int)left : each + 1) * width;
}

// A row's copy is made of 16-byte units of `each` elements that start on 16-byte boundaries.  How many elements the one takes that starts
// at `column` (below 0: in front of the row): all of them, those of neighbouring rows too, but for what is behind the tensor's end (where
// rows are narrower than a unit several end inside the last one); none where it has nothing of the row.
FDA_NORM_COPY int copied_elements(int column, int width, int each, int room) {
    if (column >= width || room == 0) return 0;
    return room - column < each ? room - column : each;
}

}  // namespace fda_norm
