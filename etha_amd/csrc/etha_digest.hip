// Digest of the sources the library was built from, in a file of its own: it changes with every source.
#include "etha_reshard.h"

#ifndef ETHA_SOURCE_HASH
#define ETHA_SOURCE_HASH "unknown"
#endif
// the marker lets a build script find the digest in the file without loading the library
static const char kSourceDigest[] = "etha-source-digest:" ETHA_SOURCE_HASH;
extern "C" const char* etha_source_hash(void) { return kSourceDigest + sizeof("etha-source-digest:") - 1; }
