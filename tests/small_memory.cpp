/* A device that runs out of memory: hipMalloc of more than a set number of
 * bytes fails, always or once, everything else is the runtime's.  Loaded with RTLD_GLOBAL
 * before the backend, whose hipMalloc is then this one. */
#include <dlfcn.h>
#include <stddef.h>

static size_t largest = ~(size_t)0, once = ~(size_t)0;

extern "C" {

/* device allocations above this many bytes fail from here on */
void small_memory(size_t bytes) { largest = bytes; }
/* the next one above this many does */
void fail_once(size_t bytes) { once = bytes; }

int hipMalloc(void **p, size_t bytes) {
    typedef int (*alloc)(void **, size_t);
    static alloc real;
    if (!real) {
        /* the one that the backend has loaded */
        const char *const names[] = {"libamdhip64.so.7", "libamdhip64.so.6",
                                     "libamdhip64.so"};
        for (const char *name : names) {
            void *runtime = real ? NULL
                                 : dlopen(name, RTLD_LAZY | RTLD_NOLOAD);
            if (runtime) real = (alloc)dlsym(runtime, "hipMalloc");
        }
        if (!real) return 1; /* hipErrorInvalidValue */
    }
    if (bytes > largest || bytes > once) {
        if (bytes > once) once = ~(size_t)0;
        *p = NULL;
        return 2; /* hipErrorOutOfMemory */
    }
    return real(p, bytes);
}

} /* extern "C" */
